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
#include <atomic>

namespace specdec {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

// What the kernels' 32-bit indexes reach: 16-row blocks of a grid's second
// dimension, offsets of 64 rows.
constexpr int64_t kLin8MaxRows = 65535 * 16, kLin8MaxFeatures = 1 << 24, kLin8MaxSteps = 1 << 16;
constexpr int64_t kLin8MaxStride = 1 << 25;

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

// More than 64 KB of LDS has to be allowed for, once a kernel and device.
template <auto Kernel> int allow_lds(int bytes) {
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return SPECDEC_EHIP;
  if (!ready[dev]) {
    if (hipFuncSetAttribute((const void *)Kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
      return SPECDEC_EHIP;
    ready[dev] = true;
  }
  return SPECDEC_OK;
}

// At most N of this wave's loads still on their way and none of its LDS
// accesses, and every wave of the workgroup here; no memory access moves across.
template <int N> __device__ __forceinline__ void wait_meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// ----------------------------------------------------------------- few rows --
constexpr int kLin8MaxWaves = 8;

// The steps of a wave: a power of two (so that four steps' scales are in one
// word), at most four waves while a wave has fewer than four steps, then at most
// eight.  Of the weight's sizes alone: the order of a row's sums does not depend
// on the other rows of the call.
inline int lin8_steps_per_wave(int steps) {
  int per = 1;
  while (per < 4 ? (steps + per - 1) / per > 4 : (steps + per - 1) / per > kLin8MaxWaves) per *= 2;
  return per;
}

// Lane l of 64's partner l ^ 8, as a rotation of each row of 16 lanes by 8.
__device__ __forceinline__ u32x4 from_partner(u32x4 v) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (unsigned)dpp_move<0x128>((int)v[i]);
  return r;
}

// The words of a row's scales that are worth LDS: see launch_lin8.
constexpr int kLin8LeastWords = 15, kLin8MostWords = 62;

__device__ __forceinline__ const __attribute__((address_space(1))) void *to_global(const uint8_t *p) {
  return (const __attribute__((address_space(1))) void *)p;
}
__device__ __forceinline__ __attribute__((address_space(3))) void *to_lds(unsigned *p) {
  return (__attribute__((address_space(3))) void *)p;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t from_corner(const uint8_t *base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, 0x7FFFFFFF, 0x00020000);
}

// 16 RT rows and F feature tiles a workgroup; the waves split the steps and
// their sums are added in wave order.  A wave asks for KB steps of W and x at
// once and there are up to 8 waves of up to 256 registers, so x, which every
// workgroup reads, comes from L2 straight to registers.  One load takes eight
// whole lines, 128 inputs of eight rows, so that no line is asked for in halves:
// lanes c < 8 of each 16 take the first halves of rows c, then c + 8, lanes c >= 8
// the second halves of rows c - 8, then c, and partners exchange what is not their
// row's.  What the L1 does most is look up x: neighbouring lanes share a look-up
// where their 16 bytes are one piece of 64, so a load of W is 16, but a load of x,
// whose neighbouring lanes hold different rows, 64 (8 where the rows are past the
// end and so one), and an unstaged load of scales 64.  Counted
// (TCP_TOTAL_CACHE_ACCESSES), 40 x 8192 x 2048: 11.4 K a workgroup, 4.1 K of them
// W's and 7.0 K x's; lanes along a row would look up a quarter of the latter.
// The loads go through buffer resources (one base and the lane's 32-bit offset), in the
// order in which the products read them, and the first word's steps stand before
// the loop: 40 x 2048 x 16384 9.2 us -> 7.8, 64 x 2048 x 16384 10.7 -> 9.6,
// 1 x 2048 x 16384 4.9 -> 4.6.
template <int RT, int F, int KB, bool STAGED>
__global__ __launch_bounds__(kLin8MaxWaves * 64) void linear_fp8_kernel(Lin8Args a) {
  extern __shared__ f32x4 s_acc[];  // [wave][RT][F][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const bool upper = c >= 8;
  const int ftiles = (a.N + 15) / 16, n0 = blockIdx.x * (16 * F);
  const int64_t m0 = (int64_t)blockIdx.y * (16 * RT);
  const int m_last = (int)min(a.M - 1 - m0, (int64_t)16 * RT - 1);
  const int s_lo = wave * a.per_wave, s_hi = min(s_lo + a.per_wave, a.steps);
  // features past N read the last tile's, rows past M the last row; neither is stored
  int wat[F];  // a tile's offset in bytes: at most 3 * 2^16 steps of 2 KB
  unsigned wsoff[F], xoff[RT][2], xsoff[RT];
  const int ws_stride = (a.steps + 3) / 4 * 4;
#pragma unroll
  for (int f = 0; f < F; ++f) {
    wat[f] = (min((int)blockIdx.x * F + f, ftiles - 1) - (int)blockIdx.x * F) * a.steps * 2048;
    wsoff[f] = (unsigned)(min(n0 + 16 * f + c, a.N - 1) - n0) * ws_stride;
  }
  const auto from_w = from_corner(a.w + (int64_t)blockIdx.x * F * a.steps * 2048);
  const uint8_t *wsb = a.ws + (int64_t)n0 * ws_stride;
  const uint8_t *xb = a.x + m0 * a.x_stride, *xsb = a.xs + m0 * a.xs_stride;
  const auto from_x = from_corner(xb), from_xs = from_corner(xsb), from_ws = from_corner(wsb);
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      xoff[t][h] = (unsigned)min(16 * t + 8 * h + (c & 7), m_last) * (unsigned)a.x_stride + (upper ? 64 : 0) + 16 * g;
    xsoff[t] = (unsigned)min(16 * t + c, m_last) * (unsigned)a.xs_stride;
  }
  // what is added before the rounding, asked for now: wave w finishes the
  // (w / F)-th 16 rows of the (w % F)-th tile
  uint16_t pre[4] = {0, 0, 0, 0};
  auto load_add = [&](int o) {
    const int row = 16 * (o / F) + c, f0 = n0 + 16 * (o % F) + 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      pre[i] = a.add[(m0 + min(row, m_last)) * a.add_stride + min(f0 + i, a.N - 1)];
  };
  if (a.add && wave < RT * F) load_add(wave);
  // the scales, a load a row: [F feature tiles, RT row tiles][16][words + 1]
  const int words = ws_stride / 4;
  unsigned *s_scales = reinterpret_cast<unsigned *>(s_acc + nw * RT * F * 64);
  if constexpr (STAGED) {
    if (lane < words) {
      for (int r = wave; r < 16 * (F + RT); r += nw) {
        const uint8_t *row = r < 16 * F ? wsb + (unsigned)(min(n0 + r, a.N - 1) - n0) * ws_stride
                                        : xsb + (unsigned)min(r - 16 * F, m_last) * (unsigned)a.xs_stride;
        __builtin_amdgcn_global_load_lds(to_global(row + 4 * lane), to_lds(s_scales + r * (words + 1)), 4, 0, 0);
      }
    }
    asm volatile("" ::: "memory");  // the loads below come behind these
    __builtin_amdgcn_sched_barrier(0);
  }
  f32x4 acc[RT][F];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int f = 0; f < F; ++f) acc[t][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  const auto quad = [&](int s4, bool first) {  // the steps of a word of scales
    const int word = s4 & ~3;
    unsigned sa[F], sb[RT];
    if constexpr (!STAGED) {
#pragma unroll
      for (int f = 0; f < F; ++f) sa[f] = __builtin_amdgcn_raw_buffer_load_b32(from_ws, wsoff[f], word, 0);
#pragma unroll
      for (int t = 0; t < RT; ++t) sb[t] = __builtin_amdgcn_raw_buffer_load_b32(from_xs, xsoff[t], word, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    const int end = min(s4 + 4, s_hi);
#pragma unroll
    for (int h = 0; h < 4; h += KB) {
      if (s4 + h < end) {
        u32x4 W[KB][F][2], X[KB][RT][2];
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          const int s = min(s4 + h + j, end - 1);
#pragma unroll
          for (int f = 0; f < F; ++f) {
            W[j][f][0] = __builtin_amdgcn_raw_buffer_load_b128(from_w, 16 * lane, wat[f] + s * 2048, 0);
            W[j][f][1] = __builtin_amdgcn_raw_buffer_load_b128(from_w, 16 * lane + 1024, wat[f] + s * 2048, 0);
          }
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              X[j][t][e] = __builtin_amdgcn_raw_buffer_load_b128(from_x, xoff[t][e], s * 128, 0);
          __builtin_amdgcn_sched_barrier(0);  // in this order, all of them before the first product
        }
        if (STAGED && h == 0) {
          // once a wave, and each has a step: its first batch stays on its way
          if (first) wait_meet<KB * 2 * (F + RT)>();
          const unsigned *at = s_scales + c * (words + 1) + (s4 >> 2);
#pragma unroll
          for (int f = 0; f < F; ++f) sa[f] = at[16 * f * (words + 1)];
#pragma unroll
          for (int t = 0; t < RT; ++t) sb[t] = at[16 * (F + t) * (words + 1)];
        }
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          const int s = s4 + h + j;
          if (s < end) {
            const int byte = 8 * (s & 3);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              const u32x4 got = from_partner(upper ? X[j][t][0] : X[j][t][1]);
              const i32x8 x = join8(upper ? got : X[j][t][0], upper ? X[j][t][1] : got);
#pragma unroll
              for (int f = 0; f < F; ++f)
                acc[t][f] = mfma8(join8(W[j][f][0], W[j][f][1]), x, acc[t][f], sa[f] >> byte, sb[t] >> byte);
            }
          }
        }
      }
    }
  };
  if constexpr (STAGED) {
    for (int s4 = s_lo; s4 < s_hi; s4 += 4) quad(s4, s4 == s_lo);
  } else {
    quad(s_lo, true);  // most waves have no more
    for (int s4 = s_lo + 4; s4 < s_hi; s4 += 4) quad(s4, false);
  }
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int f = 0; f < F; ++f) s_acc[((wave * RT + t) * F + f) * 64 + lane] = acc[t][f];
  __syncthreads();
  for (int o = wave; o < RT * F; o += nw) {
    if (a.add && o != wave) load_add(o);
    const int row = 16 * (o / F) + c, f0 = n0 + 16 * (o % F) + 4 * g;
    f32x4 v = s_acc[o * 64 + lane];
    for (int w = 1; w < nw; ++w) v += s_acc[(w * RT * F + o) * 64 + lane];
    if (row > m_last) continue;
    uint16_t *dst = a.out + (m0 + row) * a.out_stride + f0;
    uint16_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y = v[i];
      if (a.add) y += __uint_as_float((unsigned)pre[i] << 16);
      out[i] = __builtin_bit_cast(uint16_t, __float2bfloat16(y));
    }
    if (f0 + 3 < a.N) {
      __builtin_memcpy(dst, out, 8);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (f0 + i < a.N) dst[i] = out[i];
    }
  }
}

template <int RT, int F, int KB, bool STAGED> int launch_lin8(const Lin8Args &a, int waves, hipStream_t s) {
  constexpr int kScaleRows = STAGED ? 16 * (RT + F) * 4 : 0;
  constexpr int kMost = kLin8MaxWaves * RT * F * 1024 + kScaleRows * (kLin8MostWords + 1);
  static_assert(kMost <= 160 * 1024 && KB * 2 * (F + RT) < 64, "");
  const int lds = waves * RT * F * 1024 + kScaleRows * ((a.steps + 3) / 4 + 1);
  const dim3 grid((unsigned)(((a.N + 15) / 16 + F - 1) / F), (unsigned)((a.M + 16 * RT - 1) / (16 * RT)));
  if (lds > 65536) {
    const int st = allow_lds<linear_fp8_kernel<RT, F, KB, STAGED>>(kMost);
    if (st != SPECDEC_OK) return st;
  }
  linear_fp8_kernel<RT, F, KB, STAGED><<<grid, waves * 64, lds, s>>>(a);
  return launch_status();
}

// Every wave looks up the lines of its rows' scales; where there are many rows
// and many words a row, the workgroup brings them to LDS once instead.
// 40 x 8192 x 2048 (16 words a row) 9.3 us -> 8.45, 40 x 16384 x 2048 16.3 ->
// 14.3, 5 x 8192 x 2048 6.2 -> 6.1, but 1 x 8192 x 2048 5.45 -> 5.6 and
// 1 x 12288 x 2048 6.45 -> 6.9; 40 x 6144 x 2048 7.3 -> 7.25 and 16 x 7168 x 2048
// 6.75 -> 6.85 gain nothing and 40 x 5120 x 2048 6.2 -> 6.75 loses.
template <int RT, int F, int KB> int launch_lin8(const Lin8Args &call, hipStream_t s) {
  Lin8Args a = call;
  a.per_wave = lin8_steps_per_wave(a.steps);
  const int waves = (a.steps + a.per_wave - 1) / a.per_wave, words = (a.steps + 3) / 4;
  if (a.M > 4 && words >= kLin8LeastWords && words <= kLin8MostWords)
    return launch_lin8<RT, F, KB, true>(a, waves, s);
  return launch_lin8<RT, F, KB, false>(a, waves, s);
}

// The blocks of RT x F tiles, and how long a step of the fullest compute unit's
// take: 9 a tile of rows, whose loads look up the most and whose halves are
// exchanged, and 4 a tile of features.  The two numbers are fitted to the times
// at few_rows().
template <int RT, int F> inline int64_t few_cost(const Lin8Args &a, int64_t cus) {
  const int64_t blocks = (a.M + 16 * RT - 1) / (16 * RT) * ((a.N + 16 * F - 1) / (16 * F));
  return (blocks + cus - 1) / cus * (9 * RT + 4 * F);
}

// What a call runs on: rows x features of a workgroup, and how many steps of
// rows its ring in LDS holds (0: the few-row kernel, rows straight to registers).
struct Lin8Choice {
  int (*launch)(const Lin8Args &, hipStream_t);
  int rows, features, ring;
  int64_t cost;  // of the few-row kernel's blocks
};

template <int RT, int F, int KB> inline Lin8Choice few_choice(const Lin8Args &a, int64_t cus) {
  return {launch_lin8<RT, F, KB>, 16 * RT, 16 * F, 0, few_cost<RT, F>(a, cus)};
}

// The block with the least cost.  Measured, block for block (cost in brackets):
// 40 x 2048 x 16384 7.8 us with 3 x 4 (43), 8.4 with 4 x 4 (52), 8.7 with 2 x 4
// (68), 9.4 with 1 x 4 (75); 40 x 4096 x 4096 7.4 us with 1 x 4 (25), 8.7 with
// 1 x 2 (34), 9.5 with 2 x 4 (34); 40 x 8192 x 2048 8.5 us with 1 x 2 (17), 10.4
// with 1 x 4 (25), 11.1 with 1 x 1 (26); 16 x 2048 x 6144 4.0 us with 1 x 2 (17),
// 4.7 with 1 x 4 (25), 4.9 with 1 x 1 (26); 200 x 2048 x 2048 6.2 us with 2 x 4
// (34), 6.8 with 1 x 4 (50).  One tile of rows brings little beside the weight,
// and where that comes from memory (many weights in turn) the smaller blocks
// spread it better: 5 x 4096 x 14336 12.7 us with 1 x 2, 14.5 with 1 x 4, 5 x
// 2048 x 16384 8.0 and 8.5 (the same weight again and again: 4.5 with either).
// The least cost is not the least time everywhere: of one tile of rows and 8192
// features and inputs, 1 row takes 13.7 us with the 1 x 2 chosen and 12.2 with 1 x 1
// (weights from memory 16.1 and 14.6), 5 rows 13.4 and 12.6 (16.0 and 15.7), 16
// rows 13.6 and 13.2 (but 16.5 and 17.9).
// Steps asked for at once, KB: 1 against 2 8.3 and 8.5 us at 32 x 2048 x 16384, 2
// against 1 9.6 and 9.9 at 64 rows.
inline Lin8Choice few_rows(const Lin8Args &a, int64_t cus) {
  const Lin8Choice all[] = {few_choice<1, 1, 4>(a, cus), few_choice<1, 2, 4>(a, cus), few_choice<1, 4, 4>(a, cus),
                            few_choice<2, 4, 1>(a, cus), few_choice<3, 4, 1>(a, cus), few_choice<4, 4, 2>(a, cus)};
  const int choices = a.M <= 16 ? 2 : 6;
  const Lin8Choice *best = all;
  for (int i = 1; i < choices; ++i)
    if (all[i].cost < best->cost) best = &all[i];
  return *best;
}

// ---------------------------------------------------------------- many rows --
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

// The tile kernel's shape: WM x WN waves of 16 TR rows x 16 TF features, and
// its LDS: kSlotsW slots of half of the features x 128 inputs, SX of the rows x
// 128 inputs, two of 16 groups' scales; the waves' output rows (padded by 16
// bytes so that neither the 8-byte writes down a column of rows nor the 16-byte
// reads along a row meet in a bank) take their place at the end.
template <int TR, int TF, int WM, int WN, int SX> struct Tile8 {
  static_assert(WM * WN == 4 && TF % TR == 0 && TF >= 4 && TR % 2 == 0 && SX >= 3, "");
  static constexpr int kTR = TR, kTF = TF, kWM = WM, kWN = WN, kSlotsX = SX;
  // a step's rows are asked for 2 SX - 3 turns before they are read, features as
  // many at most
  static constexpr int kAhead = SX == 3 ? 2 : 2 * SX - 3, kSlotsW = kAhead + 1;
  static constexpr int kRows = 16 * TR * WM, kFeatures = 16 * TF * WN;
  static constexpr int kW = kFeatures * 64, kX = kRows * 128, kScales = (kRows + kFeatures) * 16;
  static constexpr int kXAt = kSlotsW * kW, kScalesAt = kXAt + SX * kX;
  static constexpr int kPitch = 32 * TF + 16;
  static constexpr int kRings = kScalesAt + 2 * kScales, kOut = 4 * 16 * TR * kPitch;
  static constexpr int kLds = kRings > kOut ? kRings : kOut;
  static constexpr int kLoadsW = kW / 4096, kLoadsX = kX / 8192;  // a wave's loads of a turn
  // behind the first turn's rows and features
  static constexpr int kFirst = kLoadsW * (kSlotsW - 1) + kLoadsX * (2 * SX - 3);
  static_assert(kFirst < 64, "");
  static constexpr int kPerCu = 160 * 1024 / kLds;
  static_assert(kPerCu >= 1, "");
};

// 1 KB from memory straight to LDS: lane l's 16 bytes at offset `lane_off` +
// `off` of the resource go to dst + 16 l.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, uint8_t *dst, int lane_off, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)dst, 16, lane_off, off, 0, 0);
}

// acc += w x, the operands scaled by byte K of sw and sx.  In assembly so that
// the sum stays in its registers: given the choice the compiler moves sums from
// one set to another, and a tile's take half of the register file.  Nothing in
// a turn reads a sum, so none of the hazards that the compiler would have to
// pad arises before settle().
template <int K>
__device__ __forceinline__ void product(f32x4 &acc, const i32x8 &w, const i32x8 &x, unsigned sw, unsigned sx) {
  if constexpr (K == 0)
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
                 : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
  else if constexpr (K == 1)
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0]"
                 : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
  else if constexpr (K == 2)
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0]"
                 : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
  else
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0]"
                 : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
}
// Behind the last product, before sums are read: what is still in the unit ends
// first (at most 18 cycles are asked for).
template <int TR, int TF> __device__ __forceinline__ void settle(f32x4 (&acc)[TR][TF]) {
  asm volatile("s_nop 15\n\ts_nop 15");
#pragma unroll
  for (int i = 0; i < TR; ++i)
#pragma unroll
    for (int j = 0; j < TF; j += 4)
      asm volatile("" : "+a"(acc[i][j]), "+a"(acc[i][j + 1]), "+a"(acc[i][j + 2]), "+a"(acc[i][j + 3]));
}

// A tile of kRows x kFeatures a workgroup, on v_mfma_scale_f32_16x16x128_f8f6f4
// (at this size the card's power bounds the matrix unit, and of its two shapes
// this one does more per watt: with random operands in registers 3765 TFLOP/s,
// 32x32x64 3113).  Operands go from memory straight to LDS, in instructions of
// 1 KB that touch eight whole cache lines, eight neighbouring lanes to a row (16
// look-ups in L1 each): features in the order in which they are stored, rows with the 16-byte
// chunk c of row r at place c ^ (r / 2 % 8) of its 128 bytes, so that the
// 16-byte LDS reads of either meet in no bank.  A turn multiplies 128 inputs of
// half of a wave's features with all its rows; its operands are in registers
// when it starts, the next turn's are read from LDS and later ones asked for
// between its products, so one barrier a turn is the only wait.
template <typename L, bool ADD>
__global__ __launch_bounds__(256, L::kPerCu > 2 ? 2 : L::kPerCu) void linear_fp8_tile_kernel(Lin8Args a, int tiles_m,
                                                                                             int tiles_n) {
  extern __shared__ __align__(1024) uint8_t s_ring[];
  constexpr int TR = L::kTR, TF = L::kTF, WN = L::kWN;
  constexpr int kHalf = TF / 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  // the tile: 8 XCDs take turns in the launch order, so each gets a contiguous
  // run of tiles; a run walks eight row tiles of one feature tile, then the next
  int tm, tn;
  {
    constexpr int kBand = 8;
    const int total = tiles_m * tiles_n, x = blockIdx.x % 8;
    const int t = x * (total / 8) + min(x, total % 8) + (int)blockIdx.x / 8;
    const int band = t / (kBand * tiles_n), in = t % (kBand * tiles_n);
    const int rows = min(kBand, tiles_m - band * kBand);
    tm = band * kBand + in % rows;
    tn = in / rows;
  }
  const int64_t m0 = (int64_t)tm * L::kRows;
  const int n0 = tn * L::kFeatures;
  const int wm = wave / WN, wn = wave % WN;
  const int m_last = (int)min(a.M - 1 - m0, (int64_t)L::kRows), n_last = a.N - 1 - n0;

  // this wave's share of the loads, by 32-bit offsets from the tile's corner
  // (features and rows past the ends read the last ones; they are never stored).
  // Block b of a turn's features is half b % 2 of the b / 2-th of their 16s.
  const int tile_bytes = a.steps * 2048;
  const __amdgpu_buffer_rsrc_t wb = from_corner(a.w + (int64_t)(n0 / 16) * tile_bytes);
  const __amdgpu_buffer_rsrc_t xb = from_corner(a.x + m0 * a.x_stride);
  int woff[2][L::kLoadsW], xoff[2 * L::kLoadsX];  // woff: the same in all lanes
#pragma unroll
  for (int i = 0; i < L::kLoadsW; ++i) {
    const int b = wave + 4 * i, t = b >> 1;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      woff[h][i] = min(t / kHalf * TF + h * kHalf + t % kHalf, n_last / 16) * tile_bytes + (b & 1) * 1024;
  }
#pragma unroll
  for (int i = 0; i < 2 * L::kLoadsX; ++i) {
    const int row = 8 * (wave + 4 * i) + (lane >> 3);
    xoff[i] = min(row, m_last) * (int)a.x_stride + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
  }
  const auto last = [&](int s) { return min(s, a.steps - 1); };  // past the end: never multiplied
  auto fetch_w = [&](int slot, int s, int h, int i) {
    load_to_lds(wb, s_ring + slot * L::kW + (wave + 4 * i) * 1024, lane * 16, woff[h][i] + last(s) * 2048);
  };
  auto fetch_x = [&](int slot, int s, int i) {
    load_to_lds(xb, s_ring + L::kXAt + slot * L::kX + (wave + 4 * i) * 1024, xoff[i], last(s) * 128);
  };
  // scales: 16 groups of the features, then of the rows, 16 bytes each
  constexpr int kScaleRows = (L::kRows + L::kFeatures + 255) / 256;  // a thread's
  const int words = (a.steps + 3) / 4;
  const unsigned *sp[kScaleRows];
#pragma unroll
  for (int i = 0; i < kScaleRows; ++i) {
    const int row = tid + 256 * i;
    sp[i] = reinterpret_cast<const unsigned *>(
        row < L::kFeatures ? a.ws + (int64_t)(n0 + min(row, n_last)) * (4 * words)
                           : a.xs + (m0 + min(row - L::kFeatures, m_last)) * a.xs_stride);
  }
  u32x4 sv[kScaleRows];
  auto load_scales = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i) {
      if (4 * chunk + 4 <= words) {
        __builtin_memcpy(&sv[i], sp[i] + 4 * chunk, 16);
      } else {  // the row's last words
#pragma unroll
        for (int k = 0; k < 4; ++k) sv[i][k] = sp[i][min(4 * chunk + k, words - 1)];
      }
    }
  };
  auto store_scales = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i)
      if (tid + 256 * i < L::kRows + L::kFeatures)
        *reinterpret_cast<u32x4 *>(s_ring + L::kScalesAt + (chunk & 1) * L::kScales + (tid + 256 * i) * 16) = sv[i];
  };
  unsigned sw[TF], sx[TR], sw_next[TF], sx_next[TR];
  auto read_scales = [&](int q) {  // the word of groups 4 q .. 4 q + 3
    const uint8_t *src = s_ring + L::kScalesAt + (q >> 2 & 1) * L::kScales + (q & 3) * 4;
#pragma unroll
    for (int i = 0; i < TF; ++i)
      sw_next[i] = *reinterpret_cast<const unsigned *>(src + ((wn * TF + i) * 16 + c) * 16);
#pragma unroll
    for (int i = 0; i < TR; ++i)
      sx_next[i] = *reinterpret_cast<const unsigned *>(src + (L::kFeatures + (wm * TR + i) * 16 + c) * 16);
  };
  auto next_scales = [&]() {
#pragma unroll
    for (int i = 0; i < TF; ++i) sw[i] = sw_next[i];
#pragma unroll
    for (int i = 0; i < TR; ++i) sx[i] = sx_next[i];
  };

  f32x4 acc[TR][TF];
#pragma unroll
  for (int i = 0; i < TR; ++i)
#pragma unroll
    for (int j = 0; j < TF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  i32x8 fw[2][kHalf], fx[TR];
  auto read_w = [&](int slot, int h, int t) {
    const u32x4 *v = reinterpret_cast<const u32x4 *>(s_ring + slot * L::kW + (wn * kHalf + t) * 2048 + lane * 16);
    fw[h][t] = join8(v[0], v[64]);
  };
  const int x_at = L::kXAt + (wm * TR * 16 + c) * 128, x_c0 = (g ^ (c >> 1)) * 16, x_c1 = ((4 + g) ^ (c >> 1)) * 16;
  auto read_x = [&](int slot, int i) {
    const uint8_t *src = s_ring + slot * L::kX + x_at + i * 2048;
    fx[i] = join8(*reinterpret_cast<const u32x4 *>(src + x_c0), *reinterpret_cast<const u32x4 *>(src + x_c1));
  };
  const auto after = [](int slot, int slots) { return slot == slots - 1 ? 0 : slot + 1; };
  const auto before = [](int slot, int slots) { return slot == 0 ? slots - 1 : slot - 1; };
  int ws = 0, xs = 0;  // slots of the current turn's features and step's rows
  // Turn (s, H): half H of the features in step s, whose scales are byte K of
  // the words.  The wait and barrier before it: this wave's loads for the reads
  // below have landed and its earlier reads are done, and behind the barrier
  // every wave's are.  So the next turn's features may be read and the slot of
  // this turn's loaded again, for three turns later.  The next step's rows are
  // read in turn (s, 1), each 16 behind the last product that takes the old
  // ones, the last 16 in turn (s + 1, 0), whose last products take them; their
  // slot is loaded again in turns (s + 1, 1) and (s + 2, 0), half in each.
  auto turn = [&](int s, auto k, auto half) {
    constexpr int K = decltype(k)::value, H = decltype(half)::value;
    constexpr int kLoads = L::kLoadsW + L::kLoadsX;
    wait_meet<kLoads *(L::kAhead - 1)>();
    const int ws_next = after(ws, L::kSlotsW), xs_next = after(xs, L::kSlotsX);
#pragma unroll
    for (int i = 0; i < TR; ++i) {
#pragma unroll
      for (int t = 0; t < kHalf; ++t) {
        product<K>(acc[i][H * kHalf + t], fw[H][t], fx[i], sw[H * kHalf + t], sx[i]);
        if (H == 0 && i == 0 && t == 0) read_x(xs, TR - 1);
        if (i < TR / 2 && t == (kHalf > 2 ? 1 : 0)) {
#pragma unroll
          for (int n = i * (TF / TR); n < (i + 1) * (TF / TR); ++n) read_w(ws_next, 1 - H, n);
        }
        if (t == kHalf - 2) {  // this turn's loads, spread over its products
#pragma unroll
          for (int l = i * kLoads / TR; l < (i + 1) * kLoads / TR; ++l) {
            if (l < L::kLoadsX) {
              if (H == 1)
                fetch_x(xs, s + L::kSlotsX, l);
              else
                fetch_x(before(xs, L::kSlotsX), s - 1 + L::kSlotsX, L::kLoadsX + l);
            } else {
              constexpr int A = H + L::kSlotsW;  // halves from the step's first on
              fetch_w(ws, s + A / 2, A & 1, l - L::kLoadsX);
            }
          }
        }
        if (H == 1 && i < TR - 1 && t == kHalf - 1) read_x(xs_next, i);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    ws = ws_next;
    if constexpr (H == 1) xs = xs_next;
  };
  auto step = [&](int s, auto k) {
    turn(s, k, std::integral_constant<int, 0>());
    turn(s, k, std::integral_constant<int, 1>());
  };
  // The first loads, as the turns before the first would have asked for them:
  // turn -j for features j before slot kSlotsW's, all others before those.
  load_scales(0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < 2 * L::kLoadsX; ++i) fetch_x(0, 0, i);
#pragma unroll
  for (int i = 0; i < L::kLoadsW; ++i) fetch_w(0, 0, 0, i);
#pragma unroll
  for (int i = 0; i < L::kLoadsW; ++i) fetch_w(1, 0, 1, i);
#pragma unroll
  for (int q = 2 - 2 * L::kSlotsX; q < 0; ++q) {  // the turn that would ask for part (q + 1) & 1 of a step's rows
    const int xstep = (q - ((q & 1) ? 1 : 2)) / 2 + L::kSlotsX, piece = q + L::kSlotsW;
    if (xstep >= 1) {
#pragma unroll
      for (int i = 0; i < L::kLoadsX; ++i) fetch_x(xstep, xstep, (q & 1 ? 0 : L::kLoadsX) + i);
    }
    if (piece >= 2) {
#pragma unroll
      for (int i = 0; i < L::kLoadsW; ++i) fetch_w(piece, piece / 2, piece & 1, i);
    }
  }
  store_scales(0);
  // rows and features of the first turn: everything but what follows W's second half
  wait_meet<L::kFirst>();
#pragma unroll
  for (int t = 0; t < kHalf; ++t) read_w(0, 0, t);
#pragma unroll
  for (int i = 0; i < TR - 1; ++i) read_x(0, i);
  read_scales(0);
  const int fours = a.steps / 4;
  for (int q = 0; q < fours; ++q) {
    next_scales();
    // the next 16 groups' scales: asked for at the start of these, stored in
    // the last word's turns, where two barriers follow before they are read
    if ((q & 3) == 0 && 4 * (q + 4) < a.steps) load_scales((q >> 2) + 1);
    step(4 * q, std::integral_constant<int, 0>());
    step(4 * q + 1, std::integral_constant<int, 1>());
    if ((q & 3) == 3) store_scales((q >> 2) + 1);
    step(4 * q + 2, std::integral_constant<int, 2>());
    read_scales(q + 1);
    step(4 * q + 3, std::integral_constant<int, 3>());
  }
  if (4 * fours < a.steps) {
    next_scales();
    step(4 * fours, std::integral_constant<int, 0>());
    if (4 * fours + 1 < a.steps) step(4 * fours + 1, std::integral_constant<int, 1>());
    if (4 * fours + 2 < a.steps) step(4 * fours + 2, std::integral_constant<int, 2>());
  }
  // every load has landed and every wave is through with the rings
  wait_meet<0>();
  settle(acc);
  // this lane's features of its rows to LDS, whole rows back
  uint8_t *mine = s_ring + wave * 16 * TR * L::kPitch;
  const int fbase = n0 + wn * TF * 16;
  const int64_t row0 = m0 + wm * TR * 16;
  const bool whole = m_last >= L::kRows - 1 && n_last >= L::kFeatures - 1;  // nothing of the tile past the ends
#pragma unroll
  for (int i = 0; i < TR; ++i) {
    const uint16_t *src = ADD ? a.add + min(row0 + 16 * i + c, a.M - 1) * a.add_stride : nullptr;
#pragma unroll
    for (int j = 0; j < TF; ++j) {
      const int f = 16 * j + 4 * g;
      f32x4 v = acc[i][j];
      if constexpr (ADD) {
        uint16_t r[4];
        if (whole) {
          __builtin_memcpy(r, src + fbase + f, 8);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) r[k] = src[min(fbase + f + k, a.N - 1)];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += __uint_as_float((unsigned)r[k] << 16);
      }
      const bf16x2 lo{(__bf16)v[0], (__bf16)v[1]}, hi{(__bf16)v[2], (__bf16)v[3]};
      *reinterpret_cast<u32x2 *>(mine + (16 * i + c) * L::kPitch + f * 2) =
          u32x2{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
    }
  }
  asm volatile("" ::: "memory");  // a wave reads its own rows, and its LDS accesses are done in order
  constexpr int kLanes = 2 * TF, kAtOnce = 64 / kLanes;  // lanes of a row, rows of an instruction
  const int rr0 = lane / kLanes, f0 = (lane % kLanes) * 8;
  const uint8_t *back = mine + rr0 * L::kPitch + f0 * 2;
  uint16_t *dst = a.out + (row0 + rr0) * a.out_stride + fbase + f0;
  if (whole) {
#pragma unroll
    for (int v = 0; v < 16 * TR / kAtOnce; ++v) {
      const u32x4 o = *reinterpret_cast<const u32x4 *>(back + v * kAtOnce * L::kPitch);
      __builtin_memcpy(dst + (int64_t)v * kAtOnce * a.out_stride, &o, 16);
    }
  } else {
    for (int v = 0; v < 16 * TR / kAtOnce; ++v) {
      const u32x4 o = *reinterpret_cast<const u32x4 *>(back + v * kAtOnce * L::kPitch);
      if (row0 + rr0 + v * kAtOnce >= a.M) break;
      uint16_t *to = dst + (int64_t)v * kAtOnce * a.out_stride;
      if (fbase + f0 + 8 <= a.N) {
        __builtin_memcpy(to, &o, 16);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (fbase + f0 + k < a.N) to[k] = (uint16_t)(o[k >> 1] >> (16 * (k & 1)));
      }
    }
  }
}

// The tile kernel addresses a tile's operands by 32-bit offsets.
template <typename L> bool tile8_fits(const Lin8Args &a) {
  return a.x_stride <= 0x7FFFFFFF / (L::kRows + 1) && (int64_t)a.steps * 2048 <= 0x7FFFFFFF / (L::kFeatures / 16 + 1);
}

template <typename L, bool ADD> int launch_tile8_as(const Lin8Args &a, hipStream_t s) {
  const int st = allow_lds<linear_fp8_tile_kernel<L, ADD>>(L::kLds);
  if (st != SPECDEC_OK) return st;
  const int tm = (int)((a.M + L::kRows - 1) / L::kRows), tn = (a.N + L::kFeatures - 1) / L::kFeatures;
  linear_fp8_tile_kernel<L, ADD><<<tm * tn, 256, L::kLds, s>>>(a, tm, tn);
  return launch_status();
}

template <typename L> int launch_tile8(const Lin8Args &a, hipStream_t s) {
  return a.add ? launch_tile8_as<L, true>(a, s) : launch_tile8_as<L, false>(a, s);
}

// More than 64 rows: the few-row kernel or the tile that a simple account of
// its time makes the fastest.
//   A tile shape takes, for each round of as many workgroups as the card holds,
//   a start and end and so much a step of 128 inputs (measured, us, 2048 inputs
//   unless said):
//                         workgroups          start + end, a step
//     64 x 128            1 a compute unit    2.4, 0.28   64..256 workgroups 7.5..8.2 (8192 inputs 19.9..22.5), 768 21
//     128 x 128, 7 slots  1                   2.4, 0.43   128..256 10.2..11.9 (28..31.5)
//     128 x 128, 3 slots  2                   2.0, 0.95   512 19.5, 4096 136
//     256 x 256           1                   6.0, 1.43   256 31.7 (98), 1024 117
//   which gets 65 x 2048 x 16384 (8.5 us, 12 with 128 x 128), 2048 x 8192 x 2048
//   (31.5, 42 with 64 x 128), 4096 x 2048 x 2048 (19.4, 24.5 and 27 with the
//   smallest and largest) and 4096 x 2048 x 16384 (117, 136 with 128 x 128) right.
//   The few-row kernel takes 2.6 and 0.0054 a step and unit of its cost: 128 x
//   2048 x 2048 4.8 us (tiles 7.2), 128 x 8192 x 2048 10.7 (18.7), 256 x 8192 x
//   2048 15.5 (19.5); 288 x 2048 x 2048 9.1 (7.4), 100 x 2048 x 6144 8.8 (7.4).
template <typename L> inline Lin8Choice tile_choice() {
  return {launch_tile8<L>, L::kRows, L::kFeatures, L::kSlotsX, 0};
}

inline Lin8Choice many_rows(const Lin8Args &a, int64_t cus) {
  using Small = Tile8<2, 4, 2, 2, 4>;
  using Deep = Tile8<4, 4, 2, 2, 4>;
  using Pair = Tile8<4, 4, 2, 2, 3>;
  using Large = Tile8<8, 8, 2, 2, 3>;
  const auto blocks = [&](int64_t rows, int64_t features) {
    return (a.M + rows - 1) / rows * ((a.N + features - 1) / features);
  };
  const auto cost = [&](int64_t tiles, int64_t at_once, float ends, float step) {
    return (float)((tiles + at_once - 1) / at_once) * (ends + step * (float)a.steps);
  };
  const float small = cost(blocks(64, 128), cus, 2.4f, 0.28f), deep = cost(blocks(128, 128), cus, 2.4f, 0.43f);
  const float pair = cost(blocks(128, 128), 2 * cus, 2.0f, 0.95f), large = cost(blocks(256, 256), cus, 6.0f, 1.43f);
  const float least = std::min(std::min(small, deep), std::min(pair, large));
  const Lin8Choice few = few_rows(a, cus);
  if (!tile8_fits<Large>(a) || 2.6f + 0.0054f * (float)(few.cost * a.steps) <= least) return few;
  if (large == least) return tile_choice<Large>();
  if (pair == least) return tile_choice<Pair>();
  if (deep == least) return tile_choice<Deep>();
  return tile_choice<Small>();
}

inline Lin8Choice lin8_choice(const Lin8Args &a, int64_t cus) { return a.M > 64 ? many_rows(a, cus) : few_rows(a, cus); }

}  // namespace specdec

using namespace specdec;

// The sizes of a call, checked: SPECDEC_OK and `a` filled in as far as they go.
static int lin8_sizes(int64_t rows, int64_t x_stride, int64_t x_scale_stride, int64_t in_codes, int64_t out_features,
                      Lin8Args &a) {
  if (rows < 0 || in_codes <= 0 || in_codes % kFp8Group || out_features <= 0) return SPECDEC_EINVAL;
  const int64_t steps = in_codes / kFp8Group, scale_cols = (steps + 3) / 4 * 4;
  if (rows > 1 && (x_stride < in_codes || x_scale_stride < scale_cols)) return SPECDEC_EINVAL;
  if (out_features > kLin8MaxFeatures || steps > kLin8MaxSteps || rows > kLin8MaxRows) return SPECDEC_EUNSUPPORTED;
  if (rows > 1 && (x_stride > kLin8MaxStride || x_scale_stride > kLin8MaxStride)) return SPECDEC_EUNSUPPORTED;
  a.x_stride = x_stride;
  a.xs_stride = x_scale_stride;
  a.M = rows;
  a.N = (int)out_features;
  a.steps = (int)steps;
  return SPECDEC_OK;
}

SPECDEC_API int specdec_linear_fp8(const void *x, int64_t x_stride, const void *x_scales, int64_t x_scale_stride,
                                   const void *w, const void *w_scales, int64_t rows, int64_t in_codes,
                                   int64_t out_features, const void *add, int64_t add_stride, void *out,
                                   int64_t out_stride, void *stream) {
  if (rows > 1 && (out_stride < out_features || (add && add_stride < out_features))) return SPECDEC_EINVAL;
  Lin8Args a{};
  const int st = lin8_sizes(rows, x_stride, x_scale_stride, in_codes, out_features, a);
  if (st != SPECDEC_OK || rows == 0) return st;
  if (!x || !x_scales || !w || !w_scales || !out) return SPECDEC_EINVAL;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)x_stride) & 15) return SPECDEC_EINVAL;
  if (((uintptr_t)x_scales | (uintptr_t)w_scales | (uintptr_t)x_scale_stride) & 3) return SPECDEC_EINVAL;
  if (((uintptr_t)out | (uintptr_t)add) & 1) return SPECDEC_EINVAL;
  a.x = (const uint8_t *)x;
  a.xs = (const uint8_t *)x_scales;
  a.w = (const uint8_t *)w;
  a.ws = (const uint8_t *)w_scales;
  a.out = (uint16_t *)out;
  a.out_stride = out_stride;
  a.add = (const uint16_t *)add;
  a.add_stride = add_stride;
  const int64_t cus = cu_count();
  if (cus == 0) return SPECDEC_EHIP;
  return lin8_choice(a, cus).launch(a, as_stream(stream));
}

SPECDEC_API int specdec_linear_fp8_block(int64_t rows, int64_t x_stride, int64_t in_codes, int64_t out_features,
                                         int64_t compute_units, int32_t *block) {
  if (!block || compute_units < 0 || rows <= 0) return SPECDEC_EINVAL;
  Lin8Args a{};
  const int st = lin8_sizes(rows, x_stride, kLin8MaxStride, in_codes, out_features, a);
  if (st != SPECDEC_OK) return st;
  const int64_t cus = compute_units ? compute_units : cu_count();
  if (cus == 0) return SPECDEC_EHIP;
  const Lin8Choice c = lin8_choice(a, cus);
  block[0] = c.rows;
  block[1] = c.features;
  block[2] = c.ring;
  return SPECDEC_OK;
}
