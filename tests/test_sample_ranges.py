"""The sampler's ranges over a row's values, by their own source built for the
host: a search over them ends whatever the values are (no GPU needed)."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parents[1] / "speculative-decoder_amd" / "specdec" / "csrc"
DRIVER = """
#include "sample_ranges.h"
extern "C" int bins() { return specdec::kSampleBins; }
extern "C" void ranges_of(float lo, float hi, const float *v, int n, int *out) {
  const specdec::SampleRanges r(lo, hi);
  for (int i = 0; i < n; ++i) out[i] = r.of(v[i]);
}
"""
MOST = np.finfo(np.float32).max


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    at = tmp_path_factory.mktemp("ranges")
    (at / "driver.cpp").write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O2", "-ffp-contract=off", "-shared", "-fPIC", "-D__device__=",
                    "-D__forceinline__=inline", f"-I{CSRC}", "-o", str(at / "driver.so"), str(at / "driver.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "driver.so"))
    lib.ranges_of.argtypes = [ctypes.c_float, ctypes.c_float, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    return lib


def bins_of(lib, lo, hi, v):
    out = np.full(len(v), -1, dtype=np.int32)
    lib.ranges_of(lo, hi, v.ctypes.data, len(v), out.ctypes.data)
    return out


def ends():
    """Least and largest values of a search: neighbours, denormals, both signs, the type's ends, all magnitudes."""
    one, up = np.float32(1), lambda x: np.nextafter(np.float32(x), np.float32(np.inf))
    tiny = np.float32(2.0 ** -149)
    pairs = [(0, tiny), (-tiny, 0), (-tiny, tiny), (0, 1e-40), (0, 1e-36), (0, 5.9e-36), (0, 6.1e-36), (-1e-37, 1e-37),
             (one, up(one)), (-one, up(-one)), (-MOST, MOST), (0, MOST), (-MOST, 0), (-MOST, up(-MOST)),
             (-MOST, tiny), (2.0 ** -126, up(2.0 ** -126)), (0, 2.0 ** -100), (0, up(2.0 ** -100)), (-1e30, 1e-45)]
    rng = np.random.default_rng(0)
    for _ in range(4000):
        a, b = (rng.integers(0, 2 ** 32, dtype=np.uint32).view(np.float32) for _ in range(2))
        if rng.random() < 0.5:  # near to one another
            b = np.uint32(int(a.view(np.uint32)) ^ int(rng.integers(1, 1 << int(rng.integers(1, 20))))).view(np.float32)
        if np.isfinite(a) and np.isfinite(b) and a != b:
            pairs.append((min(a, b), max(a, b)))
    return [(np.float32(a), np.float32(b)) for a, b in pairs]


def test_each_cut_parts_the_least_and_the_largest(host):
    last = host.bins() - 1
    for lo, hi in ends():
        with np.errstate(over="ignore"):
            inner = (lo * np.float32(0.5) + hi * np.linspace(0, 0.5, 99).astype(np.float32)).clip(lo, hi)
        v = np.sort(np.concatenate([[lo, hi, -MOST], inner]).astype(np.float32))[::-1].copy()
        v = v[v <= hi]
        got = bins_of(host, lo, hi, v)
        assert got.min() == 0 and got.max() == last, (lo, hi)
        assert got[0] == 0 and (got[v <= lo] == last).all(), (lo, hi)
        assert (np.diff(got) >= 0).all(), (lo, hi)  # in the values' order


def rows():
    rng = np.random.default_rng(1)
    n = 5000
    spike = np.zeros(n)
    spike[7] = 1e-40
    beside = np.zeros(n)
    beside[:9] = rng.standard_normal(9)
    beside[9] = 1e-37
    near = np.where(rng.random(n) < 0.5, np.float32(1), np.nextafter(np.float32(1), np.float32(2)))
    yield from (spike, beside, near, rng.standard_normal(n) * 1e-37, rng.standard_normal(n) * 1e-44,
                rng.standard_normal(n) * 1e30, rng.choice([-MOST, 0.0, 1e-45, MOST], n),
                np.exp(rng.uniform(-103, 88, n)) * rng.choice([-1, 1], n), np.exp(-np.arange(n) / 25.0),
                rng.integers(0, 1 << 12, n).astype(np.uint32).view(np.float32))


@pytest.mark.parametrize("row", range(10))
def test_a_search_ends_at_one_value(host, row):
    """The search's loop, into the range that holds most, the first and the last,
    each until one value is left: every pass leaves some out."""
    v = list(rows())[row].astype(np.float32)
    for pick in (lambda b: np.bincount(b).argmax(), np.min, np.max):
        left, passes = v, 0
        while left.min() != left.max():
            b = bins_of(host, left.min(), left.max(), left)
            fewer = left[b == pick(b)]
            assert 0 < len(fewer) < len(left)
            left, passes = fewer, passes + 1
        assert passes <= 40  # 2^277 values' reach, 2^10 a pass, and room
