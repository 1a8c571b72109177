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

// LDS of the tile kernel, for 64 WR rows and 64 WF features: three slots of 64
// inputs of the features, three of 128 inputs of the rows, two of 16 groups'
// scales; the waves' output rows (32 of each at a time, padded by 16 bytes so
// that neither the 8-byte writes down a column of rows nor the 16-byte reads
// along a row meet in a bank) take the rings' place at the end.
constexpr int kTileSlots = 3;
template <int WR, int WF> struct Tile8 {
  static constexpr int kW = 4 * WF * 1024, kX = 8 * WR * 1024, kScales = (WR + WF) * 1024;
  static constexpr int kXAt = kTileSlots * kW, kScalesAt = kXAt + kTileSlots * kX;
  static constexpr int kPitch = 64 * WF + 16;
  static constexpr int kRings = kScalesAt + 2 * kScales, kOut = 4 * 32 * kPitch;
  static constexpr int kLds = kRings > kOut ? kRings : kOut;
  static_assert((WR + WF) % 4 == 0, "a thread loads whole rows of scales");
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t from_corner(const uint8_t *base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, 0x7FFFFFFF, 0x00020000);
}

// 1 KB from memory straight to LDS: lane l's 16 bytes at offset `lane_off` +
// `off` of the resource go to dst + 16 l.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, uint8_t *dst, int lane_off, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)dst, 16, lane_off, off, 0, 0);
}

// At most N of this wave's loads still on their way and none of its LDS
// accesses, and every wave of the workgroup here; no memory access moves across.
template <int N> __device__ __forceinline__ void wait_meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Four waves, two by two, of 32 WR rows x 32 WF features each, on
// v_mfma_scale_f32_32x32x64_f8f6f4.  Operands go from memory straight to LDS,
// in instructions of 1 KB that touch eight whole cache lines (what bounds them
// is the lines they look up, so rows come 128 inputs at a time): features in
// the order in which they are stored, rows with the 16-byte chunk c of row r at
// place c ^ (r / 2 % 8) of its 128 bytes, so that the 16-byte LDS reads of
// either meet in no bank.  A turn multiplies 64 inputs from registers while the
// next turn's are read from LDS and later ones asked for, so one barrier a turn
// is the only wait.
template <int WR, int WF, bool ADD>
__global__ __launch_bounds__(256, 1) void linear_fp8_tile_kernel(Lin8Args a, int tiles_m, int tiles_n) {
  extern __shared__ __align__(1024) uint8_t s_ring[];
  using L = Tile8<WR, WF>;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, kh = lane >> 5;
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
  const int64_t m0 = (int64_t)tm * (64 * WR);
  const int n0 = tn * (64 * WF);
  const int wm = wave >> 1, wn = wave & 1;
  const int m_last = (int)min(a.M - 1 - m0, (int64_t)64 * WR), n_last = a.N - 1 - n0;
  const int pieces = a.steps * 2;

  // this wave's share: WF 1 KB blocks of 16 features x 64 inputs a turn, 2 WR
  // blocks of 8 rows x 128 inputs every two turns, by 32-bit offsets from the
  // tile's corner (features and rows past the ends read the last ones; they are
  // never stored)
  const int tile_bytes = a.steps * 2048;
  const __amdgpu_buffer_rsrc_t wb = from_corner(a.w + (int64_t)(n0 / 16) * tile_bytes);
  const __amdgpu_buffer_rsrc_t xb = from_corner(a.x + m0 * a.x_stride);
  int woff[WF], xoff[2 * WR];  // woff: the same in all lanes
#pragma unroll
  for (int i = 0; i < WF; ++i) woff[i] = min(wave + 4 * i, n_last / 16) * tile_bytes;
#pragma unroll
  for (int i = 0; i < 2 * WR; ++i) {
    const int row = 8 * (wave + 4 * i) + (lane >> 3);
    xoff[i] = min(row, m_last) * (int)a.x_stride + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
  }
  // inputs past the end: the last ones again, never multiplied
  auto fetch_w = [&](int slot, int piece) {
    const int off = min(piece, pieces - 1) * 1024;
#pragma unroll
    for (int i = 0; i < WF; ++i)
      load_to_lds(wb, s_ring + slot * L::kW + (wave + 4 * i) * 1024, lane * 16, woff[i] + off);
  };
  auto fetch_x = [&](int slot, int step, auto part) {  // half of this wave's rows
    const int off = min(step, a.steps - 1) * 128;
#pragma unroll
    for (int i = decltype(part)::value * WR; i < (decltype(part)::value + 1) * WR; ++i)
      load_to_lds(xb, s_ring + L::kXAt + slot * L::kX + (wave + 4 * i) * 1024, xoff[i], off);
  };
  // scales: 16 groups of 64 WF features, then of 64 WR rows, 16 bytes each
  constexpr int kScaleRows = (WR + WF) / 4;  // a thread's
  const int words = (a.steps + 3) / 4;
  const unsigned *sp[kScaleRows];
#pragma unroll
  for (int i = 0; i < kScaleRows; ++i) {
    const int row = tid + 256 * i;
    sp[i] = reinterpret_cast<const unsigned *>(
        row < 64 * WF ? a.ws + (int64_t)(n0 + min(row, n_last)) * (4 * words)
                      : a.xs + (m0 + min(row - 64 * WF, m_last)) * a.xs_stride);
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
      *reinterpret_cast<u32x4 *>(s_ring + L::kScalesAt + (chunk & 1) * L::kScales + (tid + 256 * i) * 16) = sv[i];
  };
  unsigned sw[WF], sx[WR], sw_next[WF], sx_next[WR];
  auto read_scales = [&](int q) {  // the word of groups 4 q .. 4 q + 3
    const uint8_t *src = s_ring + L::kScalesAt + (q >> 2 & 1) * L::kScales + (q & 3) * 4;
#pragma unroll
    for (int i = 0; i < WF; ++i)
      sw_next[i] = *reinterpret_cast<const unsigned *>(src + ((wn * WF + i) * 32 + r) * 16);
#pragma unroll
    for (int i = 0; i < WR; ++i)
      sx_next[i] = *reinterpret_cast<const unsigned *>(src + (64 * WF + (wm * WR + i) * 32 + r) * 16);
  };

  f32x16 acc[WR][WF];
#pragma unroll
  for (int i = 0; i < WR; ++i)
#pragma unroll
    for (int j = 0; j < WF; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  i32x8 fw[2][WF], fx[2][WR];
  const int w_at = (r >> 4) * 1024 + kh * 512 + (r & 15) * 16 + wn * WF * 2048;
  const int x_at = L::kXAt + (wm * WR * 32 + r) * 128;
  const int x_swz = (r >> 1) & 7;
  auto read = [&](int w_slot, int x_slot, auto half) {
    constexpr int H = decltype(half)::value;
    const uint8_t *src = s_ring + w_slot * L::kW + w_at;
#pragma unroll
    for (int i = 0; i < WF; ++i) {
      const u32x4 *v = reinterpret_cast<const u32x4 *>(src + i * 2048);
      fw[H][i] = join8(v[0], v[16]);
    }
    const uint8_t *xsrc = s_ring + x_slot * L::kX + x_at;
    const uint8_t *c0 = xsrc + ((4 * H + 2 * kh) ^ x_swz) * 16, *c1 = xsrc + ((4 * H + 2 * kh + 1) ^ x_swz) * 16;
#pragma unroll
    for (int i = 0; i < WR; ++i)
      fx[H][i] = join8(*reinterpret_cast<const u32x4 *>(c0 + i * 4096), *reinterpret_cast<const u32x4 *>(c1 + i * 4096));
  };
  auto after = [](int slot) { return slot == kTileSlots - 1 ? 0 : slot + 1; };
  int ws = 0, xs = 0;  // slots of the current turn's features and step's rows
  // Turn q multiplies the half H of step q / 2, whose scales are byte K of the
  // words, from registers.  The wait and barrier before it: this wave's loads
  // for turn q + 1 have landed and its reads for turn q are done, and behind
  // the barrier every wave's are.  So turn q + 1's operands may be read, and
  // the features' slot of turn q and, once both halves of a step are read, its
  // rows' slot loaded again: half the rows in this turn, half in the next.
  auto turn = [&](int q, auto k, auto half) {
    constexpr int K = decltype(k)::value, H = decltype(half)::value;
    wait_meet<WR + WF>();
    read(after(ws), H == 1 ? after(xs) : xs, std::integral_constant<int, 1 - H>());
    if constexpr (H == 1)
      fetch_x(xs, (q >> 1) + kTileSlots, std::integral_constant<int, 0>());
    else
      fetch_x(xs == 0 ? kTileSlots - 1 : xs - 1, (q >> 1) - 1 + kTileSlots, std::integral_constant<int, 1>());
    fetch_w(ws, q + kTileSlots);
#pragma unroll
    for (int i = 0; i < WR; ++i)
#pragma unroll
      for (int j = 0; j < WF; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[H][j], fx[H][i], acc[i][j], 0, 0, K, (int)sw[j],
                                                                    K, (int)sx[i]);
    // between the products: the LDS reads in the first half, then the loads
    constexpr int kHalf = WR * WF / 2, kEach = WR + WF;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                            // a product
      __builtin_amdgcn_sched_group_barrier(0x100, (2 * kEach + kHalf - 1) / kHalf, 0);  // LDS reads
    }
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x010, (kEach + kHalf - 1) / kHalf, 0);  // loads
    }
    __builtin_amdgcn_sched_barrier(0);
    ws = after(ws);
    if constexpr (H == 1) xs = after(xs);
  };
  auto step = [&](int s, auto k) {
    turn(2 * s, k, std::integral_constant<int, 0>());
    turn(2 * s + 1, k, std::integral_constant<int, 1>());
  };
  load_scales(0);
#pragma unroll
  for (int i = 0; i < kTileSlots; ++i) {
    fetch_x(i, i, std::integral_constant<int, 0>());
    // the second half of the third step's rows is asked for in turn 0
    if (i + 1 < kTileSlots) fetch_x(i, i, std::integral_constant<int, 1>());
    fetch_w(i, i);
  }
  store_scales(0);
  wait_meet<0>();
  read(0, 0, std::integral_constant<int, 0>());
  read_scales(0);
  auto next_scales = [&]() {
#pragma unroll
    for (int i = 0; i < WF; ++i) sw[i] = sw_next[i];
#pragma unroll
    for (int i = 0; i < WR; ++i) sx[i] = sx_next[i];
  };
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
  // 32 rows at a time: this lane's features of its row to LDS, whole rows back
  uint8_t *mine = s_ring + wave * 32 * L::kPitch;
  const int fbase = n0 + wn * WF * 32;
  constexpr int kLanes = 4 * WF;  // lanes of a row
  const int rr0 = lane / kLanes, f0 = (lane % kLanes) * 8;
  const bool whole = m_last >= 64 * WR - 1 && n_last >= 64 * WF - 1;  // nothing of the tile past the ends
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
        if constexpr (ADD) {
          const uint16_t *src = a.add + min(row0 + r, a.M - 1) * a.add_stride;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] += __uint_as_float((unsigned)src[min(fbase + f + k, a.N - 1)] << 16);
        }
        const bf16x2 lo{(__bf16)v[0], (__bf16)v[1]}, hi{(__bf16)v[2], (__bf16)v[3]};
        *reinterpret_cast<u32x2 *>(mine + r * L::kPitch + f * 2) =
            u32x2{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
      }
    __builtin_amdgcn_sched_barrier(0);
    uint16_t *dst = a.out + (row0 + rr0) * a.out_stride + fbase + f0;
#pragma unroll
    for (int v = 0; v < kLanes / 2; ++v) {
      const int rr = v * (64 / kLanes) + rr0;
      const u32x4 o = *reinterpret_cast<const u32x4 *>(mine + rr * L::kPitch + f0 * 2);
      if (whole || (row0 + rr < a.M && fbase + f0 + 8 <= a.N)) {
        __builtin_memcpy(dst, &o, 16);
      } else if (row0 + rr < a.M) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (fbase + f0 + k < a.N) dst[k] = (uint16_t)(o[k >> 1] >> (16 * (k & 1)));
      }
      dst += (64 / kLanes) * a.out_stride;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The tile kernel addresses a tile's operands by 32-bit offsets.
template <int WR, int WF> bool tile8_fits(const Lin8Args &a) {
  return a.x_stride <= 0x7FFFFFFF / (64 * WR + 1) && (int64_t)a.steps * 2048 <= 0x7FFFFFFF / (4 * WF + 1);
}

template <int WR, int WF, bool ADD> int launch_tile8_as(const Lin8Args &a, hipStream_t s) {
  constexpr int lds = Tile8<WR, WF>::kLds;
  static bool ready[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return SPECDEC_EHIP;
  if (!ready[dev]) {
    if (hipFuncSetAttribute((const void *)linear_fp8_tile_kernel<WR, WF, ADD>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
      return SPECDEC_EHIP;
    ready[dev] = true;
  }
  const int tm = (int)((a.M + 64 * WR - 1) / (64 * WR)), tn = (a.N + 64 * WF - 1) / (64 * WF);
  linear_fp8_tile_kernel<WR, WF, ADD><<<tm * tn, 256, lds, s>>>(a, tm, tn);
  return launch_status();
}

template <int WR, int WF> int launch_tile8(const Lin8Args &a, hipStream_t s) {
  return a.add ? launch_tile8_as<WR, WF, true>(a, s) : launch_tile8_as<WR, WF, false>(a, s);
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
  if (rows > 512 && tile8_fits<4, 4>(a)) return launch_tile8<4, 4>(a, s);
  if (rows > 64 && tile8_fits<2, 2>(a)) return launch_tile8<2, 2>(a, s);
  if (rows <= 16)
    linear_fp8_kernel<1><<<dim3(tiles, 1), waves * 64, 0, s>>>(a);
  else
    linear_fp8_kernel<4><<<dim3(tiles, (unsigned)((rows + 63) / 64)), waves * 64, 0, s>>>(a);
  return launch_status();
}
