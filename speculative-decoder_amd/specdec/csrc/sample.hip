// A token for each row of logits under temperature, top-k, top-p and min-p,
// from a given uniform, and on request the distribution it was drawn from.
//
// In the order of falling logits, ties by the lower id, with w = exp((x - max)
// / T), what is kept is the shortest of three prefixes: the first top_k; those
// with w >= min_p; the least prefix whose mass reaches top_p of the mass of the
// first top_k.  The token is the least id whose running sum of kept weights, in
// the order of ids, exceeds u times their total.
//
// A prefix of the order is a cut (x, id): every larger logit, and the equal ones
// up to that id.  No row is sorted as a whole.  One workgroup takes a row:
//   1. It reads the row once, a wave a contiguous range.  The largest logits of
//      its threads in the first part bound the k-th largest of the row from below
//      (k of them are k logits), and min_p bounds by itself; what reaches the bound
//      is collected in LDS on the way, together with the maximum and the sum of
//      weights.
//   2. The few hundred collected are ranked; running sums over them give the cuts,
//      and over their ids the token.  Most rows end here.
//   3. A nucleus of thousands of ids is found from a sample of the row and one more
//      pass; a cut that is not found so (a large top_k, thousands of equal logits)
//      by histograms of the row over 2048 ranges, of counts or of weights, and by
//      ranking the range that it falls into.
//   4. Without a cut, or past one of thousands, the sums of the waves' ranges say
//      which range the token is in, and a scan of that range which id it is.
//
// Weights and their sums are held in 64 bits: a token is a comparison of u's
// multiple of the total with a running sum of up to 2^18 weights, and in 32 bits
// about one row in a hundred of a wide distribution would get the token beside.
// Sums that atomics make are of integers, so their order does not matter: weights
// in units of 2^-52, or of 2^-45 of the largest that a range can hold.
//
// What bounds it: many greedy rows of 49152 fp32 logits the memory (512 rows 20.3
// us, a copy's rate; one row 6.4).  Otherwise one row a compute unit's vector
// instructions: the whole softmax is 37 k of them, 15 of its 22 us by their issue rate
// (4 cycles at 2.4 GHz), each one an id 0.32 us; a call of few rows leaves most
// compute units idle.  512 rows of mixed nuclei wait more than they issue (39 of 104
// us): two rows a unit, and barriers between the steps.  One row and 512 of them, us:
// the whole softmax 22 and 45, top-k 50 20 and 36, min-p 0.05 13 and 29, a nucleus of
// some ten ids 25 and 58, of some 16000 58 and 103.  Slower are rows that the first
// sample is off for (512 copies of one of 433 ids 138), bf16 rows with wide nuclei,
// which spill (66 and 114), and cuts inside thousands of equal logits, which a search
// over ids reads the row some 17 times for (one bf16 row of 128001, the cut inside
// 2000: top-k 313, a nucleus 482).
#include "common.h"
#include "sample_ranges.h"

#include <float.h>
#include <limits.h>
#include <math.h>

namespace specdec {

// a lambda that is called keeps what it captures in memory
#define SAMPLE_INLINE __attribute__((always_inline))

constexpr int kSamplePieces = 6;    // pieces of 16 bytes of a part; the next part's are in flight
constexpr int kSampleShare = 512;   // logits that a wave collects
// The largest top_k that is bounded by the threads' maxima; larger ones go by
// histograms.  One row of 49152 at 400 and 401: 27.8 and 56.6 us, 64 rows 30.7 and 58.5.
// Of 512 rows, whose workgroups have half of the maxima, 39 at 200, 109 at 300, 142 at
// 400 and 120 at 401: there histograms are the faster ones from some 330 on.
constexpr int kSampleTopK = 400;
constexpr double kSampleOff = 1.0 / (1 << 17);
constexpr int kSampleGuess = 128;   // reach the bound in the first part, for a nucleus of unknown size

struct SampleArgs {
  const void *logits;
  int64_t row_stride;
  int vocab;
  const float *u;
  float temperature, top_p, min_p;
  int32_t top_k;
  const float *temperatures, *top_ps, *min_ps;  // one a row, or null
  const int32_t *top_ks;
  int64_t *token;
  float *probs;  // [rows, vocab], or null
  int64_t probs_stride;
};

// Bits of x in an order that unsigned integers compare as floats do; both zeros are one value.
__device__ __forceinline__ unsigned sample_key(float x) {
  const unsigned b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float sample_value(unsigned key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

// a b + c with c in scalar registers: as an accumulation hipcc copies each
// coefficient to vector registers first
__device__ __forceinline__ double sample_fma(double a, double b, double c) {
  double r;
  __asm__("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}

// w[k] = 2^((e[k] - base) c) within 4e-14 relative, for powers up to 1000; at
// least 2^-1000.  2^n by the exponent's bits; 2^f, |f| <= 1/2, as 1 + f q(f), q of
// the 8th power through (2^f - 1) / f at the 9 Chebyshev points, so 2^0 is 1.  N
// side by side: the chain of one takes its latency 17 times.
template <int N> __device__ __forceinline__ void sample_weights(const float (&e)[N], double base, double c, double (&w)[N]) {
  if constexpr (N > 6) {  // .. of up to six: more at once are spilled
    constexpr int A = N / 2;
    float e1[A], e2[N - A];
    double w1[A], w2[N - A];
#pragma unroll
    for (int k = 0; k < A; ++k) e1[k] = e[k];
#pragma unroll
    for (int k = A; k < N; ++k) e2[k - A] = e[k];
    sample_weights(e1, base, c, w1);
    __builtin_amdgcn_sched_barrier(0);
    sample_weights(e2, base, c, w2);
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = k < A ? w1[k] : w2[k - A];
    return;
  }
  constexpr double magic = 6755399441055744.0;  // 1.5 2^52: n in the low bits of a sum
  double f[N];
  int n[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const double y = fmax(((double)e[k] - base) * c, -1000.0);
    const double t = y + magic;
    n[k] = (int)__double2loint(t);
    f[k] = y - (t - magic);
    w[k] = 1.0203121063391729e-07;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = sample_fma(w[k], f[k], 1.3255224878668817e-06);
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = sample_fma(w[k], f[k], 1.525268684626772e-05);
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = sample_fma(w[k], f[k], 0.00015403455852453838);
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = sample_fma(w[k], f[k], 0.0013333558179043112);
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = sample_fma(w[k], f[k], 0.009618129159402558);
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = sample_fma(w[k], f[k], 0.055504108664760424);
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = sample_fma(w[k], f[k], 0.2402265069581299);
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = sample_fma(w[k], f[k], 0.6931471805599453);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    w[k] = fma(w[k], f[k], 1.0);
    w[k] = __hiloint2double(__double2hiint(w[k]) + (n[k] << 20), __double2loint(w[k]));
  }
}
__device__ __forceinline__ double sample_weight(float v, double base, double c) {
  const float e[1] = {v};
  double w[1];
  sample_weights(e, base, c, w);
  return w[0];
}

// What is kept: larger logits, and the equal ones up to an id.
struct Cut {
  float x;
  int id;
  __device__ bool keeps(float v, int i) const { return v > x || (v == x && i <= id); }
};
__device__ __forceinline__ Cut shorter(Cut a, Cut b) {
  if (a.x != b.x) return a.x > b.x ? a : b;
  return a.id < b.id ? a : b;
}

// A row of logits as a workgroup reads it: pieces of 16 aligned bytes, wave w
// the pieces (w per + j) 64 + lane, j < per.  They come through a buffer resource,
// whose bounds stand for the row's ends: up to the 16 bytes that hold its first
// and last logit, and what is not of the row is put to -inf when it is unpacked.
template <typename T, int THREADS> struct SampleRow {
  static constexpr int EPL = 16 / sizeof(T);
  const T *x;
  int V, lead, per;  // lead: elements of the first piece that belong to the row before
  __amdgpu_buffer_rsrc_t rows;
  unsigned offset;   // of this thread's first piece
  bool infinite;     // the row has +inf: those weigh the same, the others nothing

  __device__ __forceinline__ SampleRow(const void *logits, int64_t first, int vocab) : x((const T *)logits + first), V(vocab), infinite(false) {
    lead = (int)((uintptr_t)x % 16 / sizeof(T));
    const int pieces = (lead + V + EPL - 1) / EPL;
    per = (pieces + THREADS - 1) / THREADS;
    rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(x - lead), 0, pieces * 16, 0x00020000);
    offset = ((threadIdx.x / kWave) * per * kWave + (threadIdx.x & (kWave - 1))) * 16u;
  }
  __device__ __forceinline__ int id0(int j) const { return (int)(offset / 16 + j * kWave) * EPL - lead; }  // id of the first element of piece j
  __device__ __forceinline__ u32x4 piece(int j) const {
    return __builtin_amdgcn_raw_buffer_load_b128(rows, j < per ? offset + j * (kWave * 16u) : 0xFFFFFF00u, 0, 0);
  }
  __device__ __forceinline__ float value(float v) const {
    v = fmaxf(v, -INFINITY);  // a NaN is -inf
    return infinite ? (v == INFINITY ? 0.0f : -INFINITY) : v;
  }
  __device__ __forceinline__ void unpack(u32x4 v, int j, float (&e)[EPL]) const {
#pragma unroll
    for (int k = 0; k < EPL; ++k) {
      if constexpr (sizeof(T) == 4) e[k] = fmaxf(__uint_as_float(v[k]), -INFINITY);
      else e[k] = fmaxf(__uint_as_float((k & 1) ? v[k / 2] & 0xFFFF0000u : v[k / 2] << 16), -INFINITY);
    }
    const int i = id0(j);
    if (infinite || i < 0 || i + EPL > V) {
#pragma unroll
      for (int k = 0; k < EPL; ++k) e[k] = i + k >= 0 && i + k < V ? value(e[k]) : -INFINITY;
    }
  }
  // the logit of an id of the row, or anything
  __device__ __forceinline__ float at(int i) const {
    const unsigned at = (unsigned)(lead + i) * (unsigned)sizeof(T);
    if constexpr (sizeof(T) == 4) return value(__uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows, at, 0, 0)));
    else return value(__uint_as_float((unsigned)__builtin_amdgcn_raw_buffer_load_b16(rows, at, 0, 0) << 16));
  }
  __device__ __forceinline__ void load(u32x4 (&v)[kSamplePieces], int j0) const {
#pragma unroll
    for (int k = 0; k < kSamplePieces; ++k) v[k] = piece(j0 + k);
  }
  // f(v, first piece) over this thread's pieces, a part at a time, the next one in flight
  template <typename F> __device__ __forceinline__ void parts(F &&f) const {
    u32x4 v0[kSamplePieces], v1[kSamplePieces];
    load(v0, 0);
    for (int j = 0;;) {
      load(v1, j + kSamplePieces);
      f(v0, j);
      if ((j += kSamplePieces) >= per) break;
      load(v0, j + kSamplePieces);
      f(v1, j);
      if ((j += kSamplePieces) >= per) break;
    }
  }
  // f(e, id of e[0]) over this thread's pieces, to read the row again
  template <typename F> __device__ __forceinline__ void again(F &&f) const {
#pragma unroll 1
    for (int j0 = 0; j0 < per; j0 += kSamplePieces) {
      u32x4 v[kSamplePieces];
      load(v, j0);
#pragma unroll
      for (int k = 0; k < kSamplePieces; ++k) {
        if (j0 + k >= per) break;
        float e[EPL];
        unpack(v[k], j0 + k, e);
        f(e, id0(j0 + k));
        __builtin_amdgcn_sched_barrier(0);  // one piece's 64-bit values in registers at a time
      }
    }
  }
};

template <int THREADS> struct SampleShared {
  static constexpr int WAVES = THREADS / kWave, SHARE = kSampleShare;
  uint64_t raw[WAVES][SHARE];   // as collected: the order of logits, then falling id
  uint64_t bins[kSampleBins];
  uint64_t found[THREADS];      // ranked, as many at once
  union {
    struct {
      double weight[THREADS], before[THREADS];  // of the ranked, and the sum before each
    };
    short unit[kSampleBins];
  };
  float tops[THREADS];
  double wave_d[2][WAVES];
  float wave_f[2][WAVES];
  int wave_n[WAVES];
  uint64_t sums[kWave];
  int near[kWave];
  double above;
  float bound;
  int count, token, last, keep_p, keep_q, keep_m;
  unsigned lo, hi;
};

// Reductions over the workgroup with one barrier each: a reduction's slots are
// written again two reductions later, past another barrier.
template <int THREADS> struct SampleBlock {
  static constexpr int WAVES = THREADS / kWave;
  SampleShared<THREADS> &s;
  int turn = 0;
  __device__ __forceinline__ double sum(double v) {
    v = wave_sum(v);
    turn ^= 1;
    if ((threadIdx.x & (kWave - 1)) == 0) s.wave_d[turn][threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < WAVES; ++w) v += s.wave_d[turn][w];
    return v;
  }
  __device__ __forceinline__ float max(float v) {
    v = wave_max_dpp(v);
    turn ^= 1;
    if ((threadIdx.x & (kWave - 1)) == 0) s.wave_f[turn][threadIdx.x / kWave] = v;
    __syncthreads();
    v = s.wave_f[turn][0];
    for (int w = 1; w < WAVES; ++w) v = fmaxf(v, s.wave_f[turn][w]);
    return v;
  }
  // exclusive prefix over the threads
  __device__ __forceinline__ double scan(double v) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    double x = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const double y = __shfl_up(x, o, kWave);
      if (lane >= o) x += y;
    }
    turn ^= 1;
    if (lane == kWave - 1) s.wave_d[turn][wave] = x;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < wave; ++w) before += s.wave_d[turn][w];
    double e = __shfl_up(x, 1, kWave);
    if (lane == 0) e = 0.0;
    return before + e;
  }
};

// Halves lo .. hi towards the largest bound that `want` of v (N a lane) reach.
template <int N> __device__ __forceinline__ float sample_halve(const float (&v)[N], int want) {
  float lo = FLT_MAX, hi = -FLT_MAX;
  int n = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    n += __popcll(__ballot(v[k] >= -FLT_MAX));
    lo = fminf(lo, v[k] >= -FLT_MAX ? v[k] : FLT_MAX);
    hi = fmaxf(hi, v[k]);
  }
  if (n < want) return -FLT_MAX;
  lo = -wave_max_dpp(-lo);
  hi = fminf(wave_max_dpp(hi), FLT_MAX);
#pragma unroll 1
  for (int step = 0; step < 7; ++step) {
    const float mid = 0.5f * lo + 0.5f * hi;
    int reach = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) reach += __popcll(__ballot(v[k] >= mid));
    if (reach >= want) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A bound that `want` of the threads' maxima in s.tops reach, and not many more;
// -FLT_MAX where fewer are finite.  In wave 0, of every four threads the larger
// where that leaves four times as many as are wanted.  With its barrier; the caller's
// stands between the maxima and this.
template <int THREADS> __device__ __forceinline__ float sample_bound(SampleShared<THREADS> &s, int want) {
  constexpr int N = THREADS / kWave;
  const int lane = threadIdx.x;
  if (lane < kWave) {
    float v[N], four[N / 4];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = s.tops[k * kWave + lane];
#pragma unroll
    for (int k = 0; k < N / 4; ++k) four[k] = fmaxf(fmaxf(v[4 * k], v[4 * k + 1]), fmaxf(v[4 * k + 2], v[4 * k + 3]));
    const float bound = 4 * want <= N / 4 * kWave ? sample_halve(four, want) : sample_halve(v, want);
    if (lane == 0) s.bound = bound;
  }
  __syncthreads();
  return s.bound;
}

// The other half of a pair `distance` (a power of two under 64) lanes away.
__device__ __forceinline__ uint64_t sample_partner(uint64_t v, int distance) {
  const int lo = (int)v, hi = (int)(v >> 32);
  int a, b;
  if (distance == 1) a = dpp_move<0xB1>(lo), b = dpp_move<0xB1>(hi);
  else if (distance == 2) a = dpp_move<0x4E>(lo), b = dpp_move<0x4E>(hi);
  else a = __shfl_xor(lo, distance, kWave), b = __shfl_xor(hi, distance, kWave);
  return (uint64_t)(unsigned)b << 32 | (unsigned)a;
}

// s.found[0 .. n), n <= THREADS, from the largest to the least: a bitonic network
// over the next power of two, an element a thread; pairs less than 64 apart are
// within a wave and need no barrier.
template <int THREADS> __device__ __forceinline__ uint64_t sample_sort(SampleShared<THREADS> &s, int n) {
  const int tid = threadIdx.x;
  int size = 128;
  while (size < n) size <<= 1;
  uint64_t mine = tid < n ? s.found[tid] : 0;
#pragma unroll 1
  for (int k = 2; k <= size; k <<= 1) {
    const bool down = (tid & k) == 0 || k == size;
#pragma unroll 1
    for (int j = k / 2; j >= kWave; j >>= 1) {
      __syncthreads();
      s.found[tid] = mine;
      __syncthreads();
      const uint64_t other = s.found[tid ^ j];
      mine = ((other > mine) == (down == ((tid & j) == 0))) ? other : mine;
    }
    if (tid < size) {
#pragma unroll
      for (int j = kWave / 2; j > 0; j >>= 1) {
        if (j >= k) continue;
        const uint64_t other = sample_partner(mine, j);
        mine = ((other > mine) == (down == ((tid & j) == 0))) ? other : mine;
      }
    }
  }
  __syncthreads();
  s.found[tid] = mine;
  return mine;
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(4, 4))) void sample_kernel(SampleArgs a) {
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  constexpr int EPL = 16 / sizeof(T), WAVES = THREADS / kWave, SHARE = kSampleShare;
  __shared__ SampleShared<THREADS> s;
  SampleBlock<THREADS> block{s};
  SampleRow<T, THREADS> x(a.logits, row * a.row_stride, a.vocab);
  const int V = a.vocab;

  const float t_row = a.temperatures ? a.temperatures[row] : a.temperature;
  const float p_row = a.top_ps ? a.top_ps[row] : a.top_p;
  const float m_row = a.min_ps ? a.min_ps[row] : a.min_p;
  const int k_given = a.top_ks ? a.top_ks[row] : a.top_k;
  const bool greedy = !(t_row > 0.0f);
  const int k_row = !greedy && k_given > 0 && k_given < V ? k_given : 0;
  const bool by_p = !greedy && p_row < 1.0f, by_m = !greedy && m_row > 0.0f;
  const double p = fmax((double)p_row, 0.0), m = fmin((double)m_row, 1.0);
  const double c = greedy ? 0.0 : 1.4426950408889634074 / (double)t_row;
  // powers in 32 bits: c is an fp32 number of full precision, and a difference that is
  // none is a power past all that counts
  const bool single = c > 1e-30 && c < 1e38;
  const float uu = a.u[row];
  const double u = uu > 0.0f ? (double)fminf(uu, 1.0f) : 0.0;
  float *probs = a.probs ? a.probs + row * a.probs_stride : nullptr;

  // ---- 1: the row once
  // few: some hundred logits hold the cut, as far as can be said before the row is read
  const bool few = !greedy && ((k_row > 0 && k_row <= kSampleTopK) || (k_row == 0 && (by_p || by_m)));
  const int want = k_row > 0 ? k_row : kSampleGuess;
  const bool weigh = !greedy && k_row == 0 && (by_p || !by_m);  // the sum of all weights is asked for
  float top, bound;
  double mass, base;  // this thread's weights against `base`
  int top_j;          // this thread's first piece that has its largest logit
  int collected;      // by this wave; past its share they are only counted
  const auto collect = [&](const float(&e)[EPL], int i) SAMPLE_INLINE {
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
      const uint64_t hits = __ballot(e[q] >= bound);
      const int at = collected + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(hits >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)hits, 0));
      if (e[q] >= bound && at < SHARE) s.raw[wave][at] = (uint64_t)sample_key(e[q]) << 32 | (unsigned)~(i + q);
      collected += __popcll(hits);
    }
  };
  while (true) {
    top = -INFINITY;
    bound = INFINITY;
    mass = base = 0.0;
    top_j = collected = 0;
    if (tid == 0) {
      s.token = V;
      s.last = -1;
      s.keep_p = s.keep_q = s.keep_m = 1;
    }
    x.parts([&](const u32x4(&v)[kSamplePieces], int j0) SAMPLE_INLINE {
      float part[kSamplePieces];
#pragma unroll
      for (int k = 0; k < kSamplePieces; ++k) {
        part[k] = -INFINITY;
        if (j0 + k < x.per) {
          float e[EPL];
          x.unpack(v[k], j0 + k, e);
          part[k] = e[0];
#pragma unroll
          for (int q = 1; q < EPL; ++q) part[k] = fmaxf(part[k], e[q]);
        }
        if (part[k] > top) top_j = j0 + k;
        top = fmaxf(top, part[k]);
      }
      if (j0 == 0 && (few || weigh)) {
        // weights are taken against the largest logit of the first part: 64
        // bits have room for what is larger after it
        s.tops[tid] = top;
        base = (double)block.max(top);
        if (few) bound = sample_bound(s, want);
        // the least logit of weight m is no lower than against the largest so far; a
        // top-p within a top-k needs the whole of that
        if (few && by_m && (k_row == 0 || !by_p)) bound = fmaxf(bound, (float)fmax(base + log2(m) / c, (double)-FLT_MAX));
      }
      if (few) {
#pragma unroll
        for (int k = 0; k < kSamplePieces; ++k)
          if (__any(part[k] >= bound)) {
            float e[EPL];
            x.unpack(v[k], j0 + k, e);
            collect(e, x.id0(j0 + k));
          }
      }
      if (weigh) {
#pragma unroll
        for (int k = 0; k < kSamplePieces; ++k) {
          if (j0 + k >= x.per) break;
          float e[EPL];
          x.unpack(v[k], j0 + k, e);
          if (by_p) {
            float sum = 0.0f;
#pragma unroll
            for (int q = 0; q < EPL; ++q) sum += __builtin_amdgcn_exp2f((e[q] - (float)base) * (float)c);
            mass += (double)sum;
          } else {
            double w[EPL];
            sample_weights(e, base, c, w);
#pragma unroll
            for (int q = 0; q < EPL; ++q) mass += w[q];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    });
    const float own_top = top;
    top = block.max(top);
    if (few) {
      s.tops[tid] = own_top;
      if (lane == 0) s.wave_n[wave] = collected;
    }
    if (greedy && own_top == top && top > -INFINITY && top < INFINITY) {
      float e[EPL];
      x.unpack(x.piece(top_j), top_j, e);
      int first = EPL;
#pragma unroll
      for (int q = EPL - 1; q >= 0; --q)
        if (e[q] == top) first = q;
      atomicMin(&s.token, x.id0(top_j) + first);
    }
    if (top < INFINITY) break;
    x.infinite = true;  // its largest is 0 the next time
    __syncthreads();
  }
  if (top == -INFINITY) {  // no candidate
    if (tid == 0) a.token[row] = -1;
    if (probs)
      for (int i = tid; i < V; i += THREADS) probs[i] = 0.0f;
    return;
  }
  if (greedy) {
    __syncthreads();
    const int token = s.token;
    if (tid == 0) a.token[row] = token;
    if (probs)
      for (int i = tid; i < V; i += THREADS) probs[i] = i == token ? 1.0f : 0.0f;
    return;
  }
  const double dtop = (double)top;
  // the weights of a cut's ids, of this thread
  const auto weights_within = [&](Cut cut) SAMPLE_INLINE {
    double sum = 0.0;
    x.again([&](const float(&e)[EPL], int i) SAMPLE_INLINE {
      double w[EPL];
      sample_weights(e, dtop, c, w);
#pragma unroll
      for (int q = 0; q < EPL; ++q) sum += cut.keeps(e[q], i + q) ? w[q] : 0.0;
    });
    return sum;
  };
  const Cut all_ids{-FLT_MAX, INT_MAX};
  // against the row's largest now, or again where the first part was too far from it
  // For a nucleus the sum is that of 32-bit exponentials, a third of the work: they
  // are off by 2^-23 and some 2^-23 |y| of their powers y of two, from the roundings
  // of c, the difference and the product.  The largest power is at most 40 here, and
  // what is 40 below it weighs next to nothing, so they are off by 41 2^-23 or less,
  // with their sums' roundings by less than kSampleOff (64 2^-23).  Where that leaves
  // a choice the sum is taken again in 64 bits, and at once where the largest power is
  // more or 32 bits do not hold c and the differences.
  bool sure = !by_p;
  if (weigh) {
    const double up = (base - dtop) * c;
    if (up > (by_p ? -40.0 : -900.0) && up <= 0.0 && (single || !by_p)) mass *= sample_weight((float)base, dtop, c);
    else {
      mass = weights_within(all_ids);
      sure = true;
    }
  }
  double total = weigh ? block.sum(mass) : 0.0;
  // the least logit of weight m: (x - top) c >= log2 m
  float m_bound = -FLT_MAX;
  if (by_m) {
    const double border = dtop + log2(m) / c;
    m_bound = (float)fmax(border, (double)-FLT_MAX);
    if ((double)m_bound < border) m_bound = sample_value(sample_key(m_bound) + 1);
  }

  constexpr double unit52 = 4503599627370496.0;
  // Ranks the n of s.found, with weights and the sums before each.
  const auto rank = [&](int n) SAMPLE_INLINE {
    if (n <= kWave) {  // in wave 0, by counting
      if (wave == 0) {
        const uint64_t mine = lane < n ? s.found[lane] : 0;
        int above = lane < n ? 0 : lane;
        for (int r = 0; r < n; ++r) {
          const uint64_t other = (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(mine >> 32), r) << 32 |
                                 (unsigned)__builtin_amdgcn_readlane((int)mine, r);
          above += lane < n && other > mine;
        }
        s.found[above] = mine;
        __builtin_amdgcn_wave_barrier();
        const float v = sample_value((unsigned)(s.found[lane] >> 32));
        const double w = lane < n ? sample_weight(v, dtop, c) : 0.0;
        double run = w;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
          const double y = __shfl_up(run, o, kWave);
          if (lane >= o) run += y;
        }
        const double before = __shfl_up(run, 1, kWave);
        s.weight[lane] = w;
        s.before[lane] = lane ? before : 0.0;
      }
    } else {
      const uint64_t mine = sample_sort(s, n);
      const double w = tid < n ? sample_weight(sample_value((unsigned)(mine >> 32)), dtop, c) : 0.0;
      s.before[tid] = block.scan(w);
      s.weight[tid] = w;
    }
    __syncthreads();
  };
  const auto sorted_x = [&](int r) SAMPLE_INLINE { return sample_value((unsigned)(s.found[r] >> 32)); };
  const auto sorted_id = [&](int r) SAMPLE_INLINE { return (int)~(unsigned)s.found[r]; };
  // Of the first n ranked, how many have a mass before them (with `above`) short
  // of `goal`: into `keep`, which holds 1.
  const auto short_of = [&](int n, double above, double goal, int &keep) SAMPLE_INLINE {
    for (int r = tid; r < n; r += THREADS)
      if (above + s.before[r] < goal && (r + 1 == n || above + s.before[r + 1] >= goal)) keep = r + 1;
  };

  // ---- 2: the cut among the collected
  int keep = 0;  // ranked ids kept, where the cut is among them
  if (few) {
    __syncthreads();
    // the collected that reach `bound` to s.found; their number, or more than THREADS
    const auto gather = [&]() SAMPLE_INLINE {
      const int have = s.wave_n[wave];
      const unsigned least = sample_key(bound);
      int mine = 0;
      if (have <= SHARE)
        for (int r = lane; r - lane < have; r += kWave) mine += __popcll(__ballot(r < have && (unsigned)(s.raw[wave][r] >> 32) >= least));
      else mine = THREADS + 1;
      if (lane == 0) s.near[wave] = mine;
      __syncthreads();
      int at = 0, n = 0;
      for (int w = 0; w < WAVES; ++w) {
        if (w < wave) at += s.near[w];
        n += s.near[w];
      }
      if (n <= THREADS)
        for (int r = lane; r - lane < have; r += kWave) {
          const bool in = r < have && (unsigned)(s.raw[wave][r] >> 32) >= least;
          const uint64_t hits = __ballot(in);
          if (in)
            s.found[at + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(hits >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)hits, 0))] =
                s.raw[wave][r];
          at += __popcll(hits);
        }
      __syncthreads();
      return n;
    };
    // by the maxima of the whole row the bound of a top-k is a tighter one
    if (k_row > 0) bound = fmaxf(bound, sample_bound(s, want));
    int n = gather();
    if (n > THREADS) {  // the first part was not like the rest: again, by the maxima of the whole row
      bound = sample_bound(s, want);
      collected = 0;
      x.again(collect);
      __syncthreads();
      if (lane == 0) s.wave_n[wave] = collected;
      __syncthreads();
      n = gather();
    }
    if (n <= THREADS) {
      rank(n);
      const int upto = k_row > 0 ? min(k_row, n) : n;
      const double all = s.before[upto - 1] + s.weight[upto - 1];
      if (k_row > 0) {
        total = all;
        sure = true;
      }
      const double off = sure ? 0.0 : kSampleOff;
      if (by_p) short_of(upto, 0.0, p * total * (1.0 - off), s.keep_p);
      if (by_p && !sure) short_of(upto, 0.0, p * total * (1.0 + off), s.keep_q);
      if (by_m)
        for (int r = tid; r < n; r += THREADS)
          if (sorted_x(r) >= m_bound && (r + 1 == n || sorted_x(r + 1) < m_bound)) s.keep_m = r + 1;
      __syncthreads();
      if (by_p && !sure && (s.keep_p != s.keep_q || (all >= p * total * (1.0 - off) && all < p * total * (1.0 + off)))) {
        total = block.sum(weights_within(all_ids));
        sure = true;
        if (tid == 0) s.keep_p = 1;
        __syncthreads();
        short_of(upto, 0.0, p * total, s.keep_p);
        __syncthreads();
      }
      // whether the ranked hold the cut
      if (k_row > 0 || bound <= -FLT_MAX || (by_m && bound <= m_bound) || (by_p && all >= p * total))
        keep = min(upto, min(by_p ? s.keep_p : n, by_m ? s.keep_m : n));
    }
  }

  if (keep > 0 && keep <= kWave) {
    // the token among them: the running sum up to each id, in wave 0
    if (probs)
      for (int i = tid; i < V; i += THREADS) probs[i] = 0.0f;
    total = s.before[keep - 1] + s.weight[keep - 1];
    if (wave == 0) {
      const int id = lane < keep ? sorted_id(lane) : INT_MAX;
      const double w = lane < keep ? s.weight[lane] : 0.0;
      double run = 0.0, all = 0.0;
      for (int r = 0; r < keep; ++r) {
        const int other = __builtin_amdgcn_readlane(id, r);
        const double v = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(w), r),
                                          __builtin_amdgcn_readlane(__double2loint(w), r));
        all += v;
        run += other <= id ? v : 0.0;
      }
      if (lane < keep) {
        atomicMax(&s.last, id);
        if (run > u * all) atomicMin(&s.token, id);
      }
      __builtin_amdgcn_wave_barrier();
      if (lane == 0) a.token[row] = s.token < V ? s.token : s.last;
    }
    if (probs) {
      __syncthreads();
      if (tid < keep) probs[sorted_id(tid)] = (float)(s.weight[tid] / total);
    }
    return;
  }
  if (keep > 0) {
    // the token among them: the 64th of the ids that the running sum passes the
    // goal in, then the id.  The sums are integers, so their order does not matter.
    const int shift = max(0, 26 - __clz(V));  // V >> shift < 64
    if (tid < kWave) s.sums[tid] = 0;
    if (tid == 0) s.count = 0;
    __syncthreads();
    for (int r = tid; r < keep; r += THREADS) {
      atomicAdd((unsigned long long *)&s.sums[sorted_id(r) >> shift], (unsigned long long)(s.weight[r] * unit52));
      if (u == 0.0) atomicMin(&s.token, sorted_id(r));  // the first, however little it weighs
    }
    __syncthreads();
    uint64_t upto = s.sums[lane];
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint64_t y = __shfl_up((unsigned long long)upto, o, kWave);
      if (lane >= o) upto += y;
    }
    const uint64_t whole = __shfl((unsigned long long)upto, kWave - 1, kWave);
    const double goal = u * (double)whole;
    const uint64_t past = __ballot((double)upto > goal), any = __ballot(s.sums[lane] > 0);
    const int part = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)any);
    const uint64_t first = __shfl((unsigned long long)(upto - s.sums[lane]), part, kWave);
    // that 64th's ids by themselves: of hundreds kept a few
    for (int q = tid; q < keep; q += THREADS)
      if (sorted_id(q) >> shift == part) s.bins[atomicAdd(&s.count, 1)] = q;
    __syncthreads();
    const int members = s.count;
    for (int i = tid; i < members; i += THREADS) {
      const int q = (int)s.bins[i], id = sorted_id(q);
      uint64_t run = first;
      for (int j = 0; j < members; ++j) {
        const int r = (int)s.bins[j];
        run += sorted_id(r) <= id ? (uint64_t)(s.weight[r] * unit52) : 0;
      }
      if (s.weight[q] * unit52 >= 1.0) atomicMax(&s.last, id);
      if ((double)run > goal) atomicMin(&s.token, id);
    }
    if (probs)
      for (int i = tid; i < V; i += THREADS) probs[i] = 0.0f;
    __syncthreads();
    if (tid == 0) a.token[row] = s.token < V ? s.token : s.last;
    if (probs) {
      const double inv = 1.0 / (s.before[keep - 1] + s.weight[keep - 1]);
      for (int q = tid; q < keep; q += THREADS) probs[sorted_id(q)] = (float)(s.weight[q] * inv);
    }
    return;
  }

  // ---- 3: a nucleus of thousands
  // The shortest prefix whose mass reaches `goal`, and this thread's part of that
  // mass.  A few pieces of every thread say where the cut about is: by the weight
  // below it, of which many ids have little each, so that a sample holds a like
  // share of it.  The row read once more gives the mass above that range of
  // logits and the ids in it, among which the cut is; false where it is not.
  bool crowded = false;  // more near the cut than a wave collects
  const auto nucleus = [&](Cut &cut, double margin) SAMPLE_INLINE {
    double goal = p * total;
    constexpr int PARTS = 16 / EPL;  // pieces of a thread in the sample: 16 ids
    if (x.per < 2 * PARTS || !single) return false;
    const float lo = (float)fmax(dtop - 31.7 / c, (double)-FLT_MAX);  // e^-22: what weighs less shares the last range
    if (!(lo < top)) return false;
    const float scale = (float)(kSampleBins / ((double)top - (double)lo)), c32 = (float)c;
    const auto bin_of = [&](float v) SAMPLE_INLINE { return (int)fminf((top - v) * scale, kSampleBins - 1.0f); };
    for (int q = tid; q < kSampleBins; q += THREADS) s.bins[q] = 0;
    __syncthreads();
    constexpr float unit40 = 1099511627776.0f;
    u32x4 v[PARTS];
#pragma unroll
    for (int k = 0; k < PARTS; ++k) v[k] = x.piece((2 * k + 1) * x.per / (2 * PARTS));
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
      float e[EPL];
      x.unpack(v[k], (2 * k + 1) * x.per / (2 * PARTS), e);
#pragma unroll
      for (int q = 0; q < EPL; ++q) {
        const float w = __builtin_amdgcn_exp2f((e[q] - top) * c32);
        if (e[q] >= -FLT_MAX) atomicAdd((unsigned long long *)&s.bins[bin_of(e[q])], (unsigned long long)(w * unit40));
      }
    }
    if (tid == 0) {
      s.near[0] = 0;
      s.near[1] = kSampleBins - 1;
    }
    __syncthreads();
    constexpr int N = kSampleBins / THREADS;
    double w[N], sum = 0.0;
#pragma unroll
    for (int q = 0; q < N; ++q) sum += w[q] = (double)s.bins[kSampleBins - 1 - (N * tid + q)];
    double below = block.scan(sum);  // from the least weight up
    const double aim = (total - goal) * PARTS / x.per * unit40;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int bin = kSampleBins - 1 - (N * tid + q);
      if (below < (1.0 - margin) * aim && below + w[q] >= (1.0 - margin) * aim) s.near[1] = bin;  // the range ends here
      if (below < (1.0 + margin) * aim && below + w[q] >= (1.0 + margin) * aim) s.near[0] = bin;  // .. and begins here
      below += w[q];
    }
    __syncthreads();
    // logits of bins near[0] .. near[1], and one more either way
    const float from = top - (float)(s.near[1] + 2) / scale, to = top - (float)(s.near[0] - 1) / scale;
    if (!(from < to)) return false;
    bound = from;
    collected = 0;
    mass = 0.0;
    double whole = 0.0;
    x.again([&](const float(&e)[EPL], int i) SAMPLE_INLINE {
      double w[EPL];
      sample_weights(e, dtop, c, w);
      float in[EPL];
#pragma unroll
      for (int q = 0; q < EPL; ++q) {
        whole += w[q];
        mass += e[q] > to ? w[q] : 0.0;
        in[q] = e[q] > to ? -INFINITY : e[q];
      }
      collect(in, i);
    });
    const double above = block.sum(mass);
    total = block.sum(whole);
    sure = true;
    goal = p * total;
    if (lane == 0) s.wave_n[wave] = collected;
    const int have = collected;
    // the collected by 2048 ranges again, of weights in units that the largest is 2^45 of
    const double step = ((double)to - (double)from) / kSampleBins;
    const float fine = (float)(1.0 / step);
    const auto fine_of = [&](float v) SAMPLE_INLINE { return (int)fmaxf(0.0f, fminf((to - v) * fine, kSampleBins - 1.0f)); };
    const double unit = 35184372088832.0 / sample_weight(to, dtop, c);
    for (int q = tid; q < kSampleBins; q += THREADS) s.bins[q] = 0;
    if (tid == 0) {
      s.count = 0;
      s.last = -1;
      s.token = INT_MAX;
      s.keep_p = 1;
    }
    __syncthreads();
    int most = 0;
    for (int w = 0; w < WAVES; ++w) most = max(most, s.wave_n[w]);
    crowded = most > SHARE;
    if (crowded || !(above < goal)) return false;
    const auto mine = [&](int r) SAMPLE_INLINE { return sample_value((unsigned)(s.raw[wave][r] >> 32)); };
    for (int r = lane; r < have; r += kWave) {
      const float v = mine(r);
      atomicAdd((unsigned long long *)&s.bins[fine_of(v)], (unsigned long long)(sample_weight(v, dtop, c) * unit));
    }
    __syncthreads();
    double in_bin[N];
    sum = 0.0;
#pragma unroll
    for (int q = 0; q < N; ++q) sum += in_bin[q] = (double)s.bins[N * tid + q] / unit;
    double run = above + block.scan(sum);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      // the first bin that the sum reaches the goal in; weights in whole units are short
      // by less than 2^-32 of the range's largest together
      if (run < goal && run + in_bin[q] >= goal) {
        s.token = N * tid + q;
        s.above = run;
      }
      run += in_bin[q];
    }
    __syncthreads();
    const int bin = s.token;
    if (bin == INT_MAX) return false;
    for (int r = lane; r < have; r += kWave)
      if (fine_of(mine(r)) == bin) {
        const int at = atomicAdd(&s.count, 1);
        if (at < THREADS) s.found[at] = s.raw[wave][r];
      }
    __syncthreads();
    const int n = s.count;
    if (n > THREADS) return false;
    const double before = s.above;
    rank(n);
    short_of(n, before, goal, s.keep_p);
    __syncthreads();
    cut = Cut{sorted_x(s.keep_p - 1), sorted_id(s.keep_p - 1)};
    for (int r = lane; r < have; r += kWave) {
      const float v = mine(r);
      if (cut.keeps(v, (int)~(unsigned)s.raw[wave][r])) mass += sample_weight(v, dtop, c);
    }
    return true;
  };

  // .. or any other cut, by histograms
  // The shortest prefix of the ids within `in` whose count (by_count) or mass
  // reaches `goal`.
  const auto locate = [&](bool by_count, double goal, Cut in) SAMPLE_INLINE {
    // the ranges cover lo .. hi; what weighs less than e^-30 shares the last one
    float hi = top, lo = by_count ? 0.0f : (float)fmax(dtop - 43.3 / c, (double)-FLT_MAX);
    if (by_count) {
      float least = FLT_MAX;
      x.again([&](const float(&e)[EPL], int i) SAMPLE_INLINE {
#pragma unroll
        for (int q = 0; q < EPL; ++q)
          if (e[q] >= -FLT_MAX) least = fminf(least, e[q]);
      });
      lo = -block.max(-least);
    }
    double above = 0.0;  // count or mass of what is larger than hi
    const int bits = min(45, 30 + __clz(V));  // of a weight in a bin's sum, so that V of them fit
    while (true) {
      if (lo == hi) {
        // equal logits: as many of them as it takes, in the order of ids
        const double w = by_count ? 1.0 : sample_weight(hi, dtop, c);
        const double need = fmax(1.0, ceil((goal - above) / w));
        int from = 0, to = V - 1;
        while (from < to) {  // the least id up to which there are that many
          const int mid = from + (to - from) / 2;
          int mine = 0;
          x.again([&](const float(&e)[EPL], int i) SAMPLE_INLINE {
#pragma unroll
            for (int q = 0; q < EPL; ++q) mine += e[q] == hi && i + q <= mid && in.keeps(e[q], i + q);
          });
          if (block.sum((double)mine) >= need) to = mid;
          else from = mid + 1;
        }
        return shorter(in, Cut{hi, to});
      }
      const double step = ((double)hi - (double)lo) / kSampleBins;
      const SampleRanges ranges(lo, hi);
      const auto bin_of = [&](float v) SAMPLE_INLINE { return ranges.of(v); };
      // a bin's unit is the least power of two that the largest weight it can hold is
      // below 2^bits of; what weighs less than 2^-900 is not told from nothing
      for (int q = tid; q < kSampleBins; q += THREADS) {
        s.bins[q] = 0;
        s.unit[q] = (short)((int)ceil(fmax(((double)hi - q * step - dtop) * c, -900.0)) + 2 - bits);
      }
      __syncthreads();
      x.again([&](const float(&e)[EPL], int i) SAMPLE_INLINE {
        double w[EPL];
        if (!by_count) sample_weights(e, dtop, c, w);
#pragma unroll
        for (int q = 0; q < EPL; ++q)
          if (e[q] <= hi && e[q] >= -FLT_MAX && in.keeps(e[q], i + q)) {
            const int bin = bin_of(e[q]);
            uint64_t add = 1;
            if (!by_count) {
              const double scaled = __hiloint2double(__double2hiint(w[q]) - ((int)s.unit[bin] << 20), __double2loint(w[q]));
              add = __double_as_longlong(scaled + unit52) & 0xFFFFFFFFFFFFFull;
            }
            if (add) atomicAdd((unsigned long long *)&s.bins[bin], (unsigned long long)add);
          }
      });
      __syncthreads();
      // the first bin that the running sum reaches the goal in; where it falls
      // short by a last bit of the whole, the last that holds anything
      constexpr int N = kSampleBins / THREADS;
      double w[N], sum = 0.0;
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const int bin = N * tid + q;
        w[q] = by_count ? (double)s.bins[bin] : ldexp((double)s.bins[bin], s.unit[bin]);
        sum += w[q];
      }
      double run = above + block.scan(sum);
      if (tid == 0) {
        s.count = 0;
        s.lo = 0xFFFFFFFFu;
        s.hi = 0;
        s.last = -1;
        s.token = INT_MAX;
        s.keep_p = 1;
      }
      __syncthreads();
      double before[N];
#pragma unroll
      for (int q = 0; q < N; ++q) {
        before[q] = run;
        run += w[q];
        if (w[q] > 0.0) {
          atomicMax(&s.last, N * tid + q);
          if (run >= goal) atomicMin(&s.token, N * tid + q);
        }
      }
      __syncthreads();
      const int bin = min(s.token, s.last);
#pragma unroll
      for (int q = 0; q < N; ++q)
        if (bin == N * tid + q) s.above = before[q];
      __syncthreads();
      above = s.above;
      // its logits, if they can be ranked at once
      x.again([&](const float(&e)[EPL], int i) SAMPLE_INLINE {
#pragma unroll
        for (int q = 0; q < EPL; ++q)
          if (e[q] <= hi && e[q] >= -FLT_MAX && in.keeps(e[q], i + q) && bin_of(e[q]) == bin) {
            const int at = atomicAdd(&s.count, 1);
            const unsigned key = sample_key(e[q]);
            if (at < THREADS) s.found[at] = (uint64_t)key << 32 | (unsigned)~(i + q);  // ranked: in any order
            atomicMin(&s.lo, key);
            atomicMax(&s.hi, key);
          }
      });
      __syncthreads();
      const int n = s.count;
      lo = sample_value(s.lo);
      hi = sample_value(s.hi);
      if (n <= THREADS) {
        rank(n);
        if (!by_count) short_of(n, above, goal, s.keep_p);
        __syncthreads();
        const int last = min(n, by_count ? max(1, (int)(goal - above)) : s.keep_p) - 1;
        return shorter(in, Cut{sorted_x(last), sorted_id(last)});
      }
      __syncthreads();
    }
  };
  Cut cut = all_ids;
  bool summed = weigh && !by_p;  // `mass` is that of the cut
  if (by_p && k_row == 0) {
    // four times what a sum over some half of the sample's ids is off by.  Where few ids
    // hold much of the rest it is off by more, and few are near the cut: once more with
    // room for that, before the histograms (512 rows of 49152, 142 -> 102 us; as a loop
    // over the margins it spilled, and wide rows took 115 for 103).
    constexpr double margin = THREADS == 1024 ? 0.043 : 0.06;
    summed = nucleus(cut, margin);
    if (!summed && !crowded) summed = nucleus(cut, 5 * margin);
    if (!sure) total = block.sum(weights_within(all_ids));
  }
#pragma unroll 1
  for (int turn = 0; turn < 2; ++turn) {  // top-k, then top-p within it
    const bool by_count = turn == 0;
    if (by_count ? k_row == 0 : !by_p || summed) continue;
    if (!by_count && k_row > 0) total = block.sum(weights_within(cut));
    cut = locate(by_count, by_count ? (double)k_row : p * total, cut);
    __syncthreads();
  }
  if (by_m && cut.x < m_bound) {
    cut = Cut{m_bound, INT_MAX};
    summed = false;
  }

  // ---- 4: the range of the token, then the token
  if (!summed) mass = weights_within(cut);
  __syncthreads();
  const double in_wave = wave_sum(mass);
  if (tid == 0) {
    s.token = V;
    s.last = -1;
  }
  if (lane == 0) s.weight[wave] = in_wave;
  __syncthreads();
  total = 0.0;
  for (int w = 0; w < WAVES; ++w) total += s.weight[w];
  double goal = u * total, run = 0.0;
  int range = -1, last_range = 0;
  for (int w = 0; w < WAVES; ++w) {
    const double in_w = s.weight[w];
    if (in_w > 0.0) last_range = w;
    if (range < 0 && run + in_w > goal) range = w;
    if (range < 0) run += in_w;
  }
  if (range < 0) {  // u = 1: the last id that weighs
    range = last_range;
    goal = INFINITY;
  }
  const int64_t size = (int64_t)x.per * kWave * EPL;
  const int lo = (int)max((int64_t)0, range * size - x.lead), hi = (int)min((int64_t)V, (range + 1) * size - x.lead);
  const int each = (hi - lo + THREADS - 1) / THREADS;
  const int i0 = min(hi, lo + tid * each), i1 = min(hi, i0 + each);
  constexpr int AT = 6;  // of a thread's ids at once
  const auto ids = [&](int i, double(&w)[AT]) SAMPLE_INLINE {
    float e[AT];
#pragma unroll
    for (int k = 0; k < AT; ++k) e[k] = x.at(i + k);
    sample_weights(e, dtop, c, w);
#pragma unroll
    for (int k = 0; k < AT; ++k) w[k] = i + k < i1 && cut.keeps(e[k], i + k) ? w[k] : 0.0;
  };
  double mine = 0.0, w[AT];
  for (int i = i0; i < i1; i += AT) {
    ids(i, w);
#pragma unroll
    for (int k = 0; k < AT; ++k) mine += w[k];
  }
  double at = run + block.scan(mine);
  // the threads whose ids the sum passes the goal in, or nearly: the range was chosen by
  // a sum in another order, off by up to n 2^-53 for the n <= 2^15 ids of a lane
  constexpr double near = 0x1p-36;
  if (goal == INFINITY || (at <= goal * (1.0 + near) && (at + mine) * (1.0 + near) >= goal)) {
    for (int i = i0; i < i1; i += AT) {
      if (each > AT) ids(i, w);
#pragma unroll
      for (int k = 0; k < AT; ++k) {
        at += w[k];
        if (w[k] > 0.0) {
          atomicMax(&s.last, i + k);
          if (at > goal) atomicMin(&s.token, i + k);
        }
      }
    }
  }
  __syncthreads();
  if (tid == 0) a.token[row] = s.token < V ? s.token : s.last;
  if (probs) {
    const double inv = 1.0 / total;
    x.again([&](const float(&e)[EPL], int i) SAMPLE_INLINE {
      double w[EPL];
      sample_weights(e, dtop, c, w);
#pragma unroll
      for (int q = 0; q < EPL; ++q)
        if (i + q >= 0 && i + q < V) probs[i + q] = cut.keeps(e[q], i + q) ? (float)(w[q] * inv) : 0.0f;
    });
  }
}

// A row is a compute unit's work while there are units for every row, else two share one.
template <typename T> int launch_sample(const SampleArgs &a, int64_t rows, hipStream_t s) {
  if (rows <= cu_count()) sample_kernel<T, 1024><<<(unsigned)rows, 1024, 0, s>>>(a);
  else sample_kernel<T, 512><<<(unsigned)rows, 512, 0, s>>>(a);
  return launch_status();
}

}  // namespace specdec

using namespace specdec;

SPECDEC_API int specdec_sample(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                               const float *u, float temperature, const float *temperatures, int32_t top_k,
                               const int32_t *top_ks, float top_p, const float *top_ps, float min_p,
                               const float *min_ps, int64_t *token, float *probs, int64_t probs_stride,
                               void *stream) {
  if (rows < 0 || vocab <= 0 || (rows > 1 && row_stride < vocab)) return SPECDEC_EINVAL;
  if (rows == 0) return SPECDEC_OK;
  if (!logits || !u || !token || (probs && rows > 1 && probs_stride < vocab)) return SPECDEC_EINVAL;
  if ((dtype != SPECDEC_F32 && dtype != SPECDEC_BF16) || vocab > (1 << 24) || rows > INT32_MAX)
    return SPECDEC_EUNSUPPORTED;
  SampleArgs a{logits, row_stride, (int)vocab, u, temperature, top_p, min_p, top_k, temperatures, top_ps, min_ps, top_ks,
               token, probs, probs_stride};
  if (dtype == SPECDEC_F32) return launch_sample<float>(a, rows, as_stream(stream));
  return launch_sample<__hip_bfloat16>(a, rows, as_stream(stream));
}
