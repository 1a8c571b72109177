// Projections of 8-bit rows (the format of fp8.h) by an 8-bit weight on
// gfx950's scaled MFMA:
//   out[r, n] = bf16(sum_k sx[r, k / 128] x[r, k] sw[n, k / 128] w[n, k] (+ add[r, n]))
// The weight is tiled: 16 features x 128 inputs are 2 KB, [half][lane][16]:
// lane 16 g + c of half h holds feature c's inputs 64 h + 16 g .. + 15.
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 32 codes a lane of each operand, and
// as both operands list a group's inputs in one order, which order it is does
// not matter; a lane's scale byte goes to the 32 codes it brings, and a
// group's four lanes bring the same byte.
#include "fp8.h"

#include <algorithm>
#include <type_traits>

namespace specdec {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

constexpr int kLin8MaxWaves = 8;

struct Lin8Args {
  const uint8_t *x;  // codes [M, x_stride], 128 `steps` of each row used
  int64_t x_stride;
  const uint8_t *xs;  // scales [M, xs_stride]
  int64_t xs_stride;
  const uint8_t *w;   // tiled codes
  const uint8_t *ws;  // scales [N, 4 ceil(steps / 4)]
  uint16_t *out;      // [M, out_stride] bf16
  int64_t out_stride;
  const uint16_t *add;  // [M, add_stride] bf16, or null
  int64_t add_stride;
  int64_t M;
  int N;
  int steps;     // groups of 128 inputs
  int per_wave;  // steps of a wave
};

__device__ __forceinline__ i32x8 join8(u32x4 a, u32x4 b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

__device__ __forceinline__ f32x4 mfma8(i32x8 a, i32x8 b, f32x4 c, unsigned sa, unsigned sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)sa, 0, (int)sb);
}

// out's four features f0 .. f0 + 3 of row `row`
__device__ __forceinline__ void store4(const Lin8Args &a, int64_t row, int f0, f32x4 v) {
  uint16_t *dst = a.out + row * a.out_stride + f0;
  uint16_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y = v[i];
    if (a.add && f0 + i < a.N) y += __uint_as_float((unsigned)a.add[row * a.add_stride + f0 + i] << 16);
    o[i] = __builtin_bit_cast(uint16_t, __float2bfloat16(y));
  }
  if (f0 + 3 < a.N && ((uintptr_t)dst & 7) == 0) {
    *reinterpret_cast<u32x2 *>(dst) =
        u32x2{(uint32_t)o[0] | ((uint32_t)o[1] << 16), (uint32_t)o[2] | ((uint32_t)o[3] << 16)};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f0 + i < a.N) dst[i] = o[i];
  }
}

// 16 RT rows and one feature tile a workgroup; the waves split the steps and
// their sums are added in wave order.
template <int RT> __global__ __launch_bounds__(kLin8MaxWaves * 64) void linear_fp8_kernel(Lin8Args a) {
  __shared__ f32x4 s_acc[kLin8MaxWaves][RT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * RT);
  const int s_lo = wave * a.per_wave, s_hi = min(s_lo + a.per_wave, a.steps);
  const int ws_stride = (a.steps + 3) / 4 * 4;
  const uint8_t *wp = a.w + ((int64_t)blockIdx.x * a.steps) * 2048 + lane * 16;
  const uint8_t *wsp = a.ws + (int64_t)min(n0 + c, a.N - 1) * ws_stride;
  const uint8_t *xp[RT], *xsp[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {  // rows past M read the last row, never stored
    const int64_t row = min(m0 + 16 * t + c, a.M - 1);
    xp[t] = a.x + row * a.x_stride + 16 * g;
    xsp[t] = a.xs + row * a.xs_stride;
  }
  f32x4 acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = s_lo; s < s_hi; ++s) {
    const u32x4 *wv = reinterpret_cast<const u32x4 *>(wp + (int64_t)s * 2048);
    const i32x8 av = join8(wv[0], wv[64]);
    const unsigned sa = wsp[s];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const u32x4 *xv = reinterpret_cast<const u32x4 *>(xp[t] + (int64_t)s * 128);
      acc[t] = mfma8(av, join8(xv[0], xv[4]), acc[t], sa, xsp[t][s]);
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) s_acc[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < RT; t += nw) {
    const int64_t row = m0 + 16 * t + c;
    if (row >= a.M) continue;
    f32x4 v = s_acc[0][t][lane];
    for (int w = 1; w < nw; ++w) v += s_acc[w][t][lane];
    store4(a, row, n0 + 4 * g, v);
  }
}

// ---------------------------------------------------------------- many rows --
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

// LDS bytes of the tile kernel: the ring of operand pieces, later the waves'
// output rows (32 of each, padded by 16 bytes so that neither the 8-byte
// writes down a column of rows nor the 16-byte reads along a row meet in a bank)
template <int WR, int WF> constexpr int tile8_piece() { return 4 * (WR + WF) * 1024; }
template <int WR, int WF, int RING> constexpr int tile8_lds() {
  const int ring = RING * tile8_piece<WR, WF>(), outs = 4 * 32 * (64 * WF + 16);
  return ring > outs ? ring : outs;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t from_corner(const uint8_t *base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, 0x7FFFFFFF, 0x00020000);
}

// 1 KB from memory straight to LDS: lane l's 16 bytes at offset `lane_off` +
// `off` of the resource go to dst + 16 l.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, uint8_t *dst, int lane_off, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)dst, 16, lane_off, off, 0, 0);
}

// At most N of this wave's loads still on their way and none of its LDS reads,
// and every wave of the workgroup here; no memory access moves across.
template <int N> __device__ __forceinline__ void wait_meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Four waves, two by two, of 32 WR rows x 32 WF features each, on
// v_mfma_scale_f32_32x32x64_f8f6f4.  Operands pass through LDS in pieces of 64
// inputs, loaded straight from memory into a ring of RING pieces: blocks of
// 16 rows (or features) x 64 inputs, 1 KB in the order [16 bytes of inputs]
// [row], which is how the weight is stored and what a wave's 16-byte LDS reads
// take without a bank met twice.  While a piece is multiplied from registers,
// the next one's operands are read from LDS and the piece RING ahead is asked
// for, so one barrier a piece is the only wait.
template <int WR, int WF, int RING>
__global__ __launch_bounds__(256, 1) void linear_fp8_tile_kernel(Lin8Args a, int tiles_m, int tiles_n) {
  extern __shared__ __align__(1024) uint8_t s_ring[];
  constexpr int kPiece = tile8_piece<WR, WF>();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, kh = lane >> 5;
  // the tile: 8 XCDs take turns in the launch order, so each gets a contiguous
  // run of tiles; a run walks eight row tiles of one feature tile, then the next
  const int total = tiles_m * tiles_n;
  int t = blockIdx.x;
  {
    const int per = total / 8, rest = total % 8, x = t % 8, i = t / 8;
    t = x * per + min(x, rest) + i;
  }
  int tm, tn;
  {
    constexpr int kBand = 8;
    const int band = t / (kBand * tiles_n), in = t % (kBand * tiles_n);
    const int rows = min(kBand, tiles_m - band * kBand);
    tm = band * kBand + in % rows;
    tn = in / rows;
  }
  const int64_t m0 = (int64_t)tm * (64 * WR);
  const int n0 = tn * (64 * WF);
  const int wm = wave >> 1, wn = wave & 1;
  const int pieces = a.steps * 2;

  // this lane's share of a piece: WF blocks of features, WR blocks of rows,
  // addressed by 32-bit offsets from the tile's corner (features and rows past
  // the ends read the last ones; they are never stored)
  const int ftiles = (a.N + 15) / 16;
  const int tile_bytes = a.steps * 2048;
  const __amdgpu_buffer_rsrc_t wb = from_corner(a.w + (int64_t)(n0 / 16) * tile_bytes);
  const __amdgpu_buffer_rsrc_t xb = from_corner(a.x + m0 * a.x_stride);
  int woff[WF], xoff[WR];  // woff: the same in all lanes
#pragma unroll
  for (int i = 0; i < WF; ++i) woff[i] = min(wave + 4 * i, ftiles - 1 - n0 / 16) * tile_bytes;
#pragma unroll
  for (int i = 0; i < WR; ++i)
    xoff[i] = (int)(min((int64_t)(16 * (wave + 4 * i) + (lane & 15)), a.M - 1 - m0) * a.x_stride) + (lane >> 4) * 16;
  // piece p (past the end: the last one again, never multiplied) to a slot
  auto fetch = [&](int slot, int piece) {
    const int p = min(piece, pieces - 1);
    uint8_t *dst = s_ring + slot * kPiece;
#pragma unroll
    for (int i = 0; i < WF; ++i) load_to_lds(wb, dst + (wave + 4 * i) * 1024, lane * 16, woff[i] + p * 1024);
#pragma unroll
    for (int i = 0; i < WR; ++i) load_to_lds(xb, dst + (4 * WF + wave + 4 * i) * 1024, xoff[i], p * 64);
  };
  // scales: four groups a word
  const int ws_stride = (a.steps + 3) / 4 * 4;
  const __amdgpu_buffer_rsrc_t wsb = from_corner(a.ws + (int64_t)n0 * ws_stride);
  const __amdgpu_buffer_rsrc_t xsb = from_corner(a.xs + m0 * a.xs_stride);
  int wsoff[WF], xsoff[WR];
#pragma unroll
  for (int i = 0; i < WF; ++i) wsoff[i] = min((wn * WF + i) * 32 + r, a.N - 1 - n0) * ws_stride;
#pragma unroll
  for (int i = 0; i < WR; ++i)
    xsoff[i] = (int)(min((int64_t)((wm * WR + i) * 32 + r), a.M - 1 - m0) * a.xs_stride);
  unsigned sw[WF], sx[WR], sw_next[WF], sx_next[WR];
  auto load_scales = [&](int q) {
#pragma unroll
    for (int i = 0; i < WF; ++i) sw_next[i] = __builtin_amdgcn_raw_buffer_load_b32(wsb, wsoff[i], 4 * q, 0);
#pragma unroll
    for (int i = 0; i < WR; ++i) sx_next[i] = __builtin_amdgcn_raw_buffer_load_b32(xsb, xsoff[i], 4 * q, 0);
  };

  f32x16 acc[WR][WF];
#pragma unroll
  for (int i = 0; i < WR; ++i)
#pragma unroll
    for (int j = 0; j < WF; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  i32x8 fw[2][WF], fx[2][WR];
  const int at = (r >> 4) * 1024 + kh * 512 + (r & 15) * 16;
  auto read = [&](int slot, int b) {
    const uint8_t *src = s_ring + slot * kPiece + at;
#pragma unroll
    for (int i = 0; i < WF; ++i) {
      const u32x4 *v = reinterpret_cast<const u32x4 *>(src + (wn * WF + i) * 2048);
      fw[b][i] = join8(v[0], v[16]);
    }
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      const u32x4 *v = reinterpret_cast<const u32x4 *>(src + 4 * WF * 1024 + (wm * WR + i) * 2048);
      fx[b][i] = join8(v[0], v[16]);
    }
  };
  constexpr int kLoads = WR + WF;  // a wave's loads of a piece
  // Piece q is in registers (half B of the group whose scales are byte K of
  // the words).  The wait and barrier: this wave's loads of piece q + 1 have
  // landed and its reads of piece q are done; behind the barrier every wave's
  // are.  So q + 1 may be read, and q's slot loaded again.
  auto turn = [&](int q, auto k, auto half) {
    constexpr int K = decltype(k)::value, B = decltype(half)::value;
    wait_meet<kLoads *(RING - 2)>();
    fetch(q & (RING - 1), q + RING);
    read((q + 1) & (RING - 1), 1 - B);
#pragma unroll
    for (int i = 0; i < WR; ++i)
#pragma unroll
      for (int j = 0; j < WF; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[B][j], fx[B][i], acc[i][j], 0, 0, K, (int)sw[j],
                                                                    K, (int)sx[i]);
    // the memory path's instructions between the products, not before them
#pragma unroll
    for (int i = 0; i < WR * WF; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
      __builtin_amdgcn_sched_group_barrier(0x100, (2 * kLoads + WR * WF - 1) / (WR * WF), 0);  // LDS reads
      __builtin_amdgcn_sched_group_barrier(0x010, (kLoads + WR * WF - 1) / (WR * WF), 0);      // loads
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto group = [&](int s, auto k) {
    turn(2 * s, k, std::integral_constant<int, 0>());
    turn(2 * s + 1, k, std::integral_constant<int, 1>());
  };
  load_scales(0);
#pragma unroll
  for (int p = 0; p < RING; ++p) fetch(p, p);
  wait_meet<kLoads *(RING - 1)>();
  read(0, 0);
  for (int s = 0; s < a.steps; s += 4) {
#pragma unroll
    for (int i = 0; i < WF; ++i) sw[i] = sw_next[i];
#pragma unroll
    for (int i = 0; i < WR; ++i) sx[i] = sx_next[i];
    load_scales(min(s / 4 + 1, (a.steps - 1) / 4));
    group(s, std::integral_constant<int, 0>());
    if (s + 1 < a.steps) group(s + 1, std::integral_constant<int, 1>());
    if (s + 2 < a.steps) group(s + 2, std::integral_constant<int, 2>());
    if (s + 3 < a.steps) group(s + 3, std::integral_constant<int, 3>());
  }
  // every load has landed and every wave is through with the ring
  wait_meet<0>();
  // 32 rows at a time: this lane's features of its row to LDS, whole rows back
  constexpr int kPitch = 64 * WF + 16;
  uint8_t *mine = s_ring + wave * 32 * kPitch;
  const int fbase = n0 + wn * WF * 32;
#pragma unroll
  for (int i = 0; i < WR; ++i) {
    const int64_t row0 = m0 + (wm * WR + i) * 32;
#pragma unroll
    for (int j = 0; j < WF; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int f = j * 32 + 8 * e + 4 * kh;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = acc[i][j][4 * e + k];
        if (a.add) {
          const int64_t row = min(row0 + r, a.M - 1);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] += __uint_as_float((unsigned)a.add[row * a.add_stride + min(fbase + f + k, a.N - 1)] << 16);
        }
        const bf16x2 lo{(__bf16)v[0], (__bf16)v[1]}, hi{(__bf16)v[2], (__bf16)v[3]};
        *reinterpret_cast<u32x2 *>(mine + r * kPitch + f * 2) =
            u32x2{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
      }
    __builtin_amdgcn_sched_barrier(0);
    constexpr int kLanes = 4 * WF;  // lanes of a row
#pragma unroll
    for (int v = 0; v < 32 * kLanes / 64; ++v) {
      const int rr = v * (64 / kLanes) + lane / kLanes, f = (lane % kLanes) * 8;
      const u32x4 o = *reinterpret_cast<const u32x4 *>(mine + rr * kPitch + f * 2);
      if (row0 + rr >= a.M) continue;
      uint16_t *dst = a.out + (row0 + rr) * a.out_stride + fbase + f;
      if (fbase + f + 8 <= a.N) {
        __builtin_memcpy(dst, &o, 16);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (fbase + f + k < a.N) dst[k] = (uint16_t)(o[k >> 1] >> (16 * (k & 1)));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int WR, int WF, int RING> int launch_tile8(const Lin8Args &a, hipStream_t s) {
  constexpr int lds = tile8_lds<WR, WF, RING>();
  static bool ready[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return SPECDEC_EHIP;
  if (!ready[dev]) {
    if (hipFuncSetAttribute((const void *)linear_fp8_tile_kernel<WR, WF, RING>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
      return SPECDEC_EHIP;
    ready[dev] = true;
  }
  const int tm = (int)((a.M + 64 * WR - 1) / (64 * WR)), tn = (a.N + 64 * WF - 1) / (64 * WF);
  linear_fp8_tile_kernel<WR, WF, RING><<<tm * tn, 256, lds, s>>>(a, tm, tn);
  return launch_status();
}

}  // namespace specdec

using namespace specdec;

SPECDEC_API int specdec_linear_fp8(const void *x, int64_t x_stride, const void *x_scales, int64_t x_scale_stride,
                                   const void *w, const void *w_scales, int64_t rows, int64_t in_codes,
                                   int64_t out_features, const void *add, int64_t add_stride, void *out,
                                   int64_t out_stride, void *stream) {
  if (rows < 0 || in_codes <= 0 || in_codes % kFp8Group || out_features <= 0) return SPECDEC_EINVAL;
  const int64_t steps = in_codes / kFp8Group, scale_cols = (steps + 3) / 4 * 4;
  if (rows > 1 && (x_stride < in_codes || x_scale_stride < scale_cols || out_stride < out_features ||
                   (add && add_stride < out_features)))
    return SPECDEC_EINVAL;
  if (out_features > (int64_t)1 << 24 || steps > (int64_t)1 << 16 || rows > (int64_t)1 << 20)
    return SPECDEC_EUNSUPPORTED;
  if (rows == 0) return SPECDEC_OK;
  if (!x || !x_scales || !w || !w_scales || !out) return SPECDEC_EINVAL;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)x_stride) & 15) return SPECDEC_EINVAL;
  if (((uintptr_t)x_scales | (uintptr_t)w_scales | (uintptr_t)x_scale_stride) & 3) return SPECDEC_EINVAL;
  if (((uintptr_t)out | (uintptr_t)add) & 1) return SPECDEC_EINVAL;
  Lin8Args a{(const uint8_t *)x, x_stride,   (const uint8_t *)x_scales, x_scale_stride, (const uint8_t *)w,
             (const uint8_t *)w_scales, (uint16_t *)out, out_stride, (const uint16_t *)add, add_stride, rows,
             (int)out_features, (int)steps, 0};
  const int waves = std::min<int>(kLin8MaxWaves, a.steps);
  a.per_wave = (a.steps + waves - 1) / waves;
  const unsigned tiles = (unsigned)((out_features + 15) / 16);
  hipStream_t s = as_stream(stream);
  if (rows > 512) return launch_tile8<4, 4, 4>(a, s);
  if (rows > 64) return launch_tile8<2, 2, 4>(a, s);
  if (rows <= 16)
    linear_fp8_kernel<1><<<dim3(tiles, 1), waves * 64, 0, s>>>(a);
  else
    linear_fp8_kernel<4><<<dim3(tiles, (unsigned)((rows + 63) / 64)), waves * 64, 0, s>>>(a);
  return launch_status();
}
