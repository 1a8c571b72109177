// Rows in 8 bits with a scale for each 128 values (the format of fp8.h), from
// rows as they are, from the residual addition and RMSNorm before a
// projection, and from the MLP's SiLU(gate) * up.
//
// All values stay in fp32 up to the one rounding to 8 bits; the format has
// nothing to gain from bf16 steps in between.  These kernels move bytes, at what
// a large copy does (5.2 TB/s) or near it: quantize 4096 x 2048 in bf16 5.3 us,
// 4.7 TB/s; SiLU 3001 x 8192 in bf16 23.6 us, 5.2 TB/s.  A thread takes 8
// consecutive values and the 16 lanes of a DPP row make a group, so a group's
// maximum is four lane moves and no memory, and a wave's loads and stores are
// contiguous.  Rows of any width and stride: the loads need no alignment (bf16
// rows of odd width start at odd addresses; the memory path takes a 16-byte load
// at any), only a row's last values are read one by one.
#include "fp8.h"

#include <algorithm>
#include <type_traits>

namespace specdec {

constexpr int kQuantThreads = 256;
constexpr int kPer = 8;  // values a thread holds of one group

// 8 values of a row from column i on, zeros past dim
template <typename T> struct alignas(sizeof(T)) Eight {
  T v[kPer];
};
template <typename T> __device__ __forceinline__ void load8(const T *row, int64_t i, int64_t dim, float (&v)[kPer]) {
  if (i + kPer <= dim) {
    Eight<T> raw;
    __builtin_memcpy(&raw, row + i, sizeof(raw));
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = to_f32(raw.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = i + j < dim ? to_f32(row[i + j]) : 0.0f;
  }
}

// The codes and scale of the group that the calling 16 lanes hold: lane r of
// them (0 .. 15) has the values 8 r .. 8 r + 7.  `pad`: scales behind this one
// that the row's last group also writes.
__device__ __forceinline__ void store_group(const float (&y)[kPer], int r, uint8_t *codes, uint8_t *scale, int pad) {
  float m = 0.0f;  // fmaxf leaves NaN out; infinities, which are rare, are left out by a second look
#pragma unroll
  for (int j = 0; j < kPer; ++j) m = fmaxf(m, fabsf(y[j]));
  if (__any(m == INFINITY)) {
    m = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) m = fmaxf(m, fabsf(y[j]) == INFINITY ? 0.0f : fabsf(y[j]));
  }
  const unsigned byte = fp8_scale_byte(__float_as_uint(row16_max(m)));
  const float inv = fp8_inverse(byte);
  const uint2 c = make_uint2(fp8_pack4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv),
                             fp8_pack4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv));
  *reinterpret_cast<uint2 *>(codes + kPer * r) = c;
  if (r <= pad) scale[r] = (uint8_t)(r == 0 ? byte : kFp8ScaleOne);
}

// SiLU(g) * u = g / (1 + e^-g) * u in fp32 for g >= kSiluFar, as exactly as with a
// library's exp and a division (each about half a unit) and in half of their
// instructions, which would take longer than the rows' bytes (3001 x 8192 in
// bf16: 31.2 us with them).  e^-g is 2^t on the hardware's exp2, t = -g log2 e in
// two parts of which the small one is applied after; the quotient is g times the
// hardware's reciprocal with one correction by its remainder.  From g = 88.5 on
// e^-g adds nothing to 1.  Infinite gates give NaN, a code's NaN as well as an
// infinity's.
constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.92596303e-8f, kLn2 = 0.693147182f;
constexpr float kSiluFar = -80.0f;

__device__ __forceinline__ float silu_mul_f32(float g, float u) {
#pragma clang fp contract(off)
  const float x = __builtin_amdgcn_fmed3f(g, -88.5f, 88.5f);
  const float t = -x * kLog2e;
  const float low = fmaf(-x, kLog2eLow, fmaf(-x, kLog2e, -t));
  const float e0 = __builtin_amdgcn_exp2f(t);
  const float d = 1.0f + fmaf(e0, low * kLn2, e0);
  const float r = __builtin_amdgcn_rcpf(d);
  const float s0 = g * r;
  return fmaf(fmaf(-d, s0, g), r, s0) * u;
}

// The same for g < kSiluFar, rare in a model's rows.  1 + e^g is 1 there, so
// SiLU(g) = g e^g, which falls below fp32's normal values (and whose 1 + e^-g
// passes fp32) while its product with a large u is well inside: e^g = 2^k 2^f,
// and of 2^k only what keeps g e^g normal comes before u.  Below -200 the product
// is under 2^-152 with any u, a zero code as at -200.
__device__ __forceinline__ float silu_mul_far(float g, float u) {
#pragma clang fp contract(off)
  const float x = fmaxf(g, -200.0f);
  const float t = x * kLog2e;
  const float low = fmaf(x, kLog2eLow, fmaf(x, kLog2e, -t));
  const float k = rintf(t);
  const float e0 = __builtin_amdgcn_exp2f(t - k);
  const int all = (int)k, first = max(all, -120);
  const float s = ldexpf(x * fmaf(e0, low * kLn2, e0), first);
  return fmaf(0.0f, g, ldexpf(s * u, all - first));  // 0 * g: NaN for g = -inf, as -inf / inf
}

// One group for every 16 lanes; SILU: rows hold gate then up, `dim` each.
template <typename T, bool SILU>
__global__ __launch_bounds__(kQuantThreads) void quantize_kernel(const T *__restrict__ x, int64_t stride, int64_t dim,
                                                                 unsigned groups, unsigned total, uint8_t *codes,
                                                                 uint8_t *scales) {
  const unsigned id = (blockIdx.x * kQuantThreads + threadIdx.x) >> 4;
  if (id >= total) return;  // whole rows of 16 lanes
  const unsigned row = id / groups, grp = id - row * groups;
  const int r = threadIdx.x & 15;
  const T *src = x + (int64_t)row * stride;
  const int64_t i = (int64_t)grp * kFp8Group + kPer * r;
  float y[kPer];
  load8(src, i, dim, y);
  if constexpr (SILU) {
    float u[kPer];
    load8(src + dim, i, dim, u);
    // the most negative gate: among negative values the largest as bits
    unsigned least = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) least = max(least, __float_as_uint(y[j]));
    float v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = silu_mul_f32(y[j], u[j]);
    if (least > __float_as_uint(kSiluFar)) {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (y[j] < kSiluFar) v[j] = silu_mul_far(y[j], u[j]);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) y[j] = v[j];
  }
  const int64_t cols = (int64_t)groups * kFp8Group, gcols = fp8_scale_cols(dim);
  const int pad = grp + 1 == groups ? (int)(gcols - groups) : 0;
  store_group(y, r, codes + row * cols + (int64_t)grp * kFp8Group, scales + row * gcols + grp, pad);
}

// LANES threads a row (several rows a workgroup below 256), CH groups of every
// 16 lanes in registers (dim <= 8 CH LANES).  summed = round(hidden + delta), or
// hidden alone without delta; then y = summed * rsqrt(mean(summed^2) + eps) *
// weight in fp32.  The row's sum is taken in an order that dim alone fixes, so a
// row has the same bits whatever rows come with it.
// `summed` may be hidden or delta itself: the thread that writes a value has read
// it from both.
// One group of 8 values a thread and a whole row at once, as far as a workgroup
// reaches: a row's time is one round trip to memory and one sum.  4096 x 2048 in
// bf16 with the sum written 12.1 us (4.8 TB/s, what a large copy does is 5.2;
// 128 threads with two groups 13.0, 64 with four 13.2), one row 2.8 us (3.5, 4.7).
constexpr int kNormMaxLanes = 1024, kNormMaxCh = 2;

template <typename T, int CH, int LANES>
__global__ __launch_bounds__(LANES < kQuantThreads ? kQuantThreads : LANES) void add_rmsnorm_quant_kernel(
    const T *hidden, const T *delta, const T *__restrict__ weight, T *summed, int64_t rows, int64_t dim, float eps,
    unsigned groups, uint8_t *codes, uint8_t *scales) {
#pragma clang fp contract(off)
  constexpr int kThreads = LANES < kQuantThreads ? kQuantThreads : LANES;
  __shared__ float red[kThreads / kWave];
  const int64_t row = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int tid = threadIdx.x % LANES, r = tid & 15;
  if (LANES <= kWave && row >= rows) return;  // whole waves, and no barrier below
  const int64_t at = min(row, rows - 1) * dim;
  const T *h = hidden + at;
  float y[CH][kPer];
#pragma unroll
  for (int k = 0; k < CH; ++k) load8(h, (int64_t)kPer * (tid + k * LANES), dim, y[k]);
  if (delta) {
    const T *dl = delta + at;
    T *out = summed + at;
    float d[CH][kPer];
#pragma unroll
    for (int k = 0; k < CH; ++k) load8(dl, (int64_t)kPer * (tid + k * LANES), dim, d[k]);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int64_t i = (int64_t)kPer * (tid + k * LANES);
      Eight<T> s;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        s.v[j] = from_f32<T>(y[k][j] + d[k][j]);
        y[k][j] = to_f32(s.v[j]);
      }
      if (row >= rows) continue;
      if (i + kPer <= dim) {
        __builtin_memcpy(out + i, &s, sizeof(s));
      } else {
        for (int j = 0; j < kPer && i + j < dim; ++j) out[i + j] = s.v[j];
      }
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < CH; ++k)
#pragma unroll
    for (int j = 0; j < kPer; ++j) ss += y[k][j] * y[k][j];
  ss = wave_sum_dpp(ss);
  if constexpr (LANES > kWave) {
    const int first = threadIdx.x / LANES * (LANES / kWave);
    if ((tid & (kWave - 1)) == 0) red[threadIdx.x / kWave] = ss;
    __syncthreads();
    ss = red[first];
#pragma unroll
    for (int w = 1; w < LANES / kWave; ++w) ss += red[first + w];
  }
  const float inv = rsqrtf(ss / (float)dim + eps);
  const int64_t cols = (int64_t)groups * kFp8Group, gcols = fp8_scale_cols(dim);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const unsigned grp = (unsigned)(tid + k * LANES) >> 4;
    if (grp >= groups || row >= rows) break;  // whole rows of 16 lanes
    const int64_t i = (int64_t)grp * kFp8Group + kPer * r;
    float w[kPer];
    load8(weight, i, dim, w);
#pragma unroll
    for (int j = 0; j < kPer; ++j) y[k][j] = i + j < dim ? y[k][j] * inv * w[j] : 0.0f;  // 0 * inv may be NaN
    const int pad = grp + 1 == groups ? (int)(gcols - groups) : 0;
    store_group(y[k], r, codes + row * cols + (int64_t)grp * kFp8Group, scales + row * gcols + grp, pad);
  }
}

// Grid of a call of rows * groups groups, 16 lanes each; false where it passes
// what one launch's indices hold.
inline bool quant_grid(int64_t rows, int64_t groups, unsigned &total, unsigned &blocks) {
  if (groups > (int64_t)1 << 24 || rows > ((int64_t)1 << 27) / groups) return false;
  total = (unsigned)(rows * groups);
  blocks = (total + kQuantThreads / 16 - 1) / (kQuantThreads / 16);
  return true;
}

template <typename T, bool SILU>
int launch_quantize(const void *x, int64_t rows, int64_t dim, int64_t stride, uint8_t *codes, uint8_t *scales,
                    hipStream_t s) {
  const int64_t groups = (dim + kFp8Group - 1) / kFp8Group;
  unsigned total, blocks;
  if (!quant_grid(rows, groups, total, blocks)) return SPECDEC_EUNSUPPORTED;
  quantize_kernel<T, SILU><<<blocks, kQuantThreads, 0, s>>>((const T *)x, stride, dim, (unsigned)groups, total, codes,
                                                            scales);
  return launch_status();
}

template <typename T, int CH, int LANES>
int launch_add_rmsnorm_as(const void *hidden, const void *delta, const void *weight, void *summed, int64_t rows,
                          int64_t dim, float eps, uint8_t *codes, uint8_t *scales, hipStream_t s) {
  constexpr int threads = LANES < kQuantThreads ? kQuantThreads : LANES, at_once = threads / LANES;
  const int64_t blocks = (rows + at_once - 1) / at_once;
  if (blocks > UINT32_MAX / threads) return SPECDEC_EUNSUPPORTED;  // a launch holds fewer than 2^32 threads
  add_rmsnorm_quant_kernel<T, CH, LANES><<<(unsigned)blocks, threads, 0, s>>>(
      (const T *)hidden, (const T *)delta, (const T *)weight, (T *)summed, rows, dim, eps,
      (unsigned)((dim + kFp8Group - 1) / kFp8Group), codes, scales);
  return launch_status();
}

template <typename T>
int launch_add_rmsnorm_quant(const void *hidden, const void *delta, const void *weight, void *summed, int64_t rows,
                             int64_t dim, float eps, uint8_t *codes, uint8_t *scales, hipStream_t s) {
  const auto run = [&](auto ch, auto lanes) {
    return launch_add_rmsnorm_as<T, decltype(ch)::value, decltype(lanes)::value>(hidden, delta, weight, summed, rows,
                                                                                 dim, eps, codes, scales, s);
  };
  using std::integral_constant;
  const integral_constant<int, 1> one;
  if (dim <= 512) return run(one, integral_constant<int, 64>());
  if (dim <= 1024) return run(one, integral_constant<int, 128>());
  if (dim <= 2048) return run(one, integral_constant<int, 256>());
  if (dim <= 4096) return run(one, integral_constant<int, 512>());
  if (dim <= 8192) return run(one, integral_constant<int, kNormMaxLanes>());
  return run(integral_constant<int, kNormMaxCh>(), integral_constant<int, kNormMaxLanes>());
}

}  // namespace specdec

using namespace specdec;

static bool quant_out_ok(const void *codes, const void *scales) {
  return codes && scales && ((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 3) == 0;
}

SPECDEC_API int specdec_quantize_fp8(const void *x, int dtype, int64_t rows, int64_t dim, int64_t row_stride,
                                     void *codes, void *scales, void *stream) {
  if (rows < 0 || dim <= 0 || (rows > 1 && row_stride < dim)) return SPECDEC_EINVAL;
  if (dtype != SPECDEC_BF16 && dtype != SPECDEC_F32) return SPECDEC_EINVAL;
  if (rows == 0) return SPECDEC_OK;
  if (!x || !quant_out_ok(codes, scales)) return SPECDEC_EINVAL;
  uint8_t *c = (uint8_t *)codes, *sc = (uint8_t *)scales;
  return dtype == SPECDEC_BF16
             ? launch_quantize<__hip_bfloat16, false>(x, rows, dim, row_stride, c, sc, as_stream(stream))
             : launch_quantize<float, false>(x, rows, dim, row_stride, c, sc, as_stream(stream));
}

SPECDEC_API int specdec_silu_mul_fp8(const void *gate_up, int dtype, int64_t rows, int64_t inter, int64_t row_stride,
                                     void *codes, void *scales, void *stream) {
  if (rows < 0 || inter <= 0 || (rows > 1 && row_stride < 2 * inter)) return SPECDEC_EINVAL;
  if (dtype != SPECDEC_BF16 && dtype != SPECDEC_F32) return SPECDEC_EINVAL;
  if (rows == 0) return SPECDEC_OK;
  if (!gate_up || !quant_out_ok(codes, scales)) return SPECDEC_EINVAL;
  uint8_t *c = (uint8_t *)codes, *sc = (uint8_t *)scales;
  return dtype == SPECDEC_BF16
             ? launch_quantize<__hip_bfloat16, true>(gate_up, rows, inter, row_stride, c, sc, as_stream(stream))
             : launch_quantize<float, true>(gate_up, rows, inter, row_stride, c, sc, as_stream(stream));
}

SPECDEC_API int specdec_add_rmsnorm_fp8(const void *hidden, const void *delta, const void *weight, void *summed,
                                        int dtype, int64_t rows, int64_t dim, float eps, void *codes, void *scales,
                                        void *stream) {
  if (rows < 0 || dim <= 0) return SPECDEC_EINVAL;
  if (dtype != SPECDEC_BF16 && dtype != SPECDEC_F32) return SPECDEC_EINVAL;
  if (dim > (int64_t)kNormMaxLanes * kPer * kNormMaxCh || rows > UINT32_MAX) return SPECDEC_EUNSUPPORTED;
  if (rows == 0) return SPECDEC_OK;
  if (!hidden || !weight || (delta && !summed) || !quant_out_ok(codes, scales)) return SPECDEC_EINVAL;
  uint8_t *c = (uint8_t *)codes, *sc = (uint8_t *)scales;
  return dtype == SPECDEC_BF16 ? launch_add_rmsnorm_quant<__hip_bfloat16>(hidden, delta, weight, summed, rows, dim,
                                                                          eps, c, sc, as_stream(stream))
                               : launch_add_rmsnorm_quant<float>(hidden, delta, weight, summed, rows, dim, eps, c, sc,
                                                                 as_stream(stream));
}
