// Rows in 8 bits with a scale for each 128 values (the format of fp8.h), from
// rows as they are, from the residual addition and RMSNorm before a
// projection, and from the MLP's SiLU(gate) * up.
//
// All values stay in fp32 up to the one rounding to 8 bits; the format has
// nothing to gain from bf16 steps in between.  These kernels move bytes: a
// thread takes 8 consecutive values, the 16 lanes of a DPP row make a group,
// so the group's maximum is four lane moves and no memory, and a wave's loads
// and stores are contiguous.  Rows of any width and stride: the loads need no
// alignment (bf16 rows of odd width start at odd addresses; the memory path
// takes a 16-byte load at any), only a row's last values are read one by one.
#include "fp8.h"

#include <algorithm>

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
// them (0 .. 15) has the values 8 r .. 8 r + 7.  `last`: the row's last group,
// whose lanes also write the padding scales behind it.
__device__ __forceinline__ void store_group(const float (&y)[kPer], int r, uint8_t *codes, uint8_t *scale, int pad) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) m = max(m, fp8_finite_bits(y[j]));
  const unsigned byte = fp8_scale_byte(row16_max(m));
  const float inv = fp8_inverse(byte);
  const uint2 c = make_uint2(fp8_pack4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv),
                             fp8_pack4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv));
  *reinterpret_cast<uint2 *>(codes + kPer * r) = c;
  if (r <= pad) scale[r] = (uint8_t)(r == 0 ? byte : kFp8ScaleOne);
}

// SiLU(g) * u in fp32: g / (1 + e^-g) * u, each step rounded on its own.
__device__ __forceinline__ float silu_mul_f32(float g, float u) {
#pragma clang fp contract(off)
  return g / (1.0f + expf(-g)) * u;
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
#pragma unroll
    for (int j = 0; j < kPer; ++j) y[j] = silu_mul_f32(y[j], u[j]);
  }
  const int64_t cols = (int64_t)groups * kFp8Group, gcols = fp8_scale_cols(dim);
  const int pad = grp + 1 == groups ? (int)(gcols - groups) : 0;
  store_group(y, r, codes + row * cols + (int64_t)grp * kFp8Group, scales + row * gcols + grp, pad);
}

// One workgroup a row, CH groups of every 16 lanes in registers (dim <= 2048
// CH).  summed = round(hidden + delta), or hidden alone without delta; then
// y = summed * rsqrt(mean(summed^2) + eps) * weight in fp32.  The row's sum is
// taken in an order that dim alone fixes, so a row has the same bits whatever
// rows come with it.
constexpr int kNormMaxCh = 8;

template <typename T, int CH>
__global__ __launch_bounds__(kQuantThreads) void add_rmsnorm_quant_kernel(
    const T *hidden, const T *__restrict__ delta, const T *__restrict__ weight, T *summed, int64_t dim, float eps,
    unsigned groups, uint8_t *codes, uint8_t *scales) {
#pragma clang fp contract(off)
  __shared__ float red[kQuantThreads / kWave];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, r = tid & 15, lanes = blockDim.x;
  const T *h = hidden + row * dim;
  float y[CH][kPer];
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int64_t i = (int64_t)kPer * (tid + k * lanes);
    load8(h, i, dim, y[k]);
  }
  if (delta) {
    const T *dl = delta + row * dim;
    T *out = summed + row * dim;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int64_t i = (int64_t)kPer * (tid + k * lanes);
      float d[kPer];
      load8(dl, i, dim, d);
      Eight<T> s;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        s.v[j] = from_f32<T>(y[k][j] + d[j]);
        y[k][j] = to_f32(s.v[j]);
      }
      if (i + kPer <= dim) {
        __builtin_memcpy(out + i, &s, sizeof(s));
      } else {
        for (int j = 0; j < kPer && i + j < dim; ++j) out[i + j] = s.v[j];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < CH; ++k)
#pragma unroll
    for (int j = 0; j < kPer; ++j) ss += y[k][j] * y[k][j];
  ss = wave_sum_dpp(ss);
  if ((tid & (kWave - 1)) == 0) red[tid / kWave] = ss;
  __syncthreads();
  ss = red[0];
  for (int w = 1; w < lanes / kWave; ++w) ss += red[w];
  const float inv = rsqrtf(ss / (float)dim + eps);
  const int64_t cols = (int64_t)groups * kFp8Group, gcols = fp8_scale_cols(dim);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const unsigned grp = (unsigned)(tid + k * lanes) >> 4;
    if (grp >= groups) break;  // whole rows of 16 lanes
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

template <typename T>
int launch_add_rmsnorm_quant(const void *hidden, const void *delta, const void *weight, void *summed, int64_t rows,
                             int64_t dim, float eps, uint8_t *codes, uint8_t *scales, hipStream_t s) {
  const unsigned groups = (unsigned)((dim + kFp8Group - 1) / kFp8Group);
  const unsigned chunks = groups * 16;  // threads that hold one chunk each
  const dim3 grid((unsigned)rows), block(std::min<unsigned>((chunks + kWave - 1) / kWave * kWave, kQuantThreads));
  const unsigned ch = (chunks + block.x - 1) / block.x;
  const T *h = (const T *)hidden, *d = (const T *)delta, *w = (const T *)weight;
  T *o = (T *)summed;
  if (ch <= 1)
    add_rmsnorm_quant_kernel<T, 1><<<grid, block, 0, s>>>(h, d, w, o, dim, eps, groups, codes, scales);
  else if (ch <= 2)
    add_rmsnorm_quant_kernel<T, 2><<<grid, block, 0, s>>>(h, d, w, o, dim, eps, groups, codes, scales);
  else if (ch <= 4)
    add_rmsnorm_quant_kernel<T, 4><<<grid, block, 0, s>>>(h, d, w, o, dim, eps, groups, codes, scales);
  else
    add_rmsnorm_quant_kernel<T, kNormMaxCh><<<grid, block, 0, s>>>(h, d, w, o, dim, eps, groups, codes, scales);
  return launch_status();
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
  if (dim > (int64_t)kQuantThreads * kPer * kNormMaxCh || rows > INT32_MAX) return SPECDEC_EUNSUPPORTED;
  if (rows == 0) return SPECDEC_OK;
  if (!hidden || !weight || (delta && !summed) || !quant_out_ok(codes, scales)) return SPECDEC_EINVAL;
  uint8_t *c = (uint8_t *)codes, *sc = (uint8_t *)scales;
  return dtype == SPECDEC_BF16 ? launch_add_rmsnorm_quant<__hip_bfloat16>(hidden, delta, weight, summed, rows, dim,
                                                                          eps, c, sc, as_stream(stream))
                               : launch_add_rmsnorm_quant<float>(hidden, delta, weight, summed, rows, dim, eps, c, sc,
                                                                 as_stream(stream));
}
