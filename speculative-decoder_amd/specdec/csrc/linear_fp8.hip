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
  if (rows <= 16)
    linear_fp8_kernel<1><<<dim3(tiles, 1), waves * 64, 0, s>>>(a);
  else
    linear_fp8_kernel<4><<<dim3(tiles, (unsigned)((rows + 63) / 64)), waves * 64, 0, s>>>(a);
  return launch_status();
}
