// A token for each row of logits under temperature, top-k, top-p and min-p,
// from a given uniform, and on request the distribution it was drawn from.
//
// In the order of falling logits, ties by the lower id, with w = exp((x - max)
// / T), what is kept is the shortest of three prefixes: the first top_k; those
// with w >= min_p; the least prefix whose mass reaches top_p of the mass of the
// first top_k.  The token is the least id whose running sum of kept weights, in
// the order of ids, exceeds u times their total.
//
// A prefix of the order is a cut (key, ties): every id whose key is higher, and
// the first `ties` of those that have it, the key being the logit's bits in an
// order that integers compare.  So no row is sorted: a cut is found by halving
// the range of keys, counting (top-k) or adding up weights (top-p) above the
// middle.
//
// Weights and their sums are held in 64 bits: a token is a comparison of u's
// multiple of the total with a running sum of up to 2^18 weights, and in 32 bits
// about one row in a hundred of a wide distribution would get the token beside.
#include "common.h"

#include <math.h>

namespace specdec {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / kWave;

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

// Bits of x in an order that unsigned integers compare as floats do; both zeros
// are one value, a NaN is -inf.
constexpr unsigned kKeyNegInf = 0x007FFFFFu;  // the key of -inf
__device__ __forceinline__ unsigned sample_key(float x) {
  if (x != x) return kKeyNegInf;
  const unsigned b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float sample_value(unsigned key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

// w of the value with this key; the largest weighs 1 whatever it is (+inf too)
__device__ __forceinline__ double sample_weight(unsigned key, unsigned top, double inv_t) {
  if (key == top) return 1.0;
  const double d = (double)sample_value(key) - (double)sample_value(top);
  return d > -INFINITY ? exp(d * inv_t) : 0.0;
}

struct Cut {
  unsigned key;
  int ties;
};
__device__ __forceinline__ Cut shorter(Cut a, Cut b) {
  if (a.key != b.key) return a.key > b.key ? a : b;
  return a.ties < b.ties ? a : b;
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1);
  const T *x = (const T *)a.logits + row * a.row_stride;
  const int V = a.vocab;
  __shared__ double dscratch[kSampleWaves + 1];
  __shared__ int iscratch[kSampleWaves + 1];
  __shared__ int found;

  const float t_row = a.temperatures ? a.temperatures[row] : a.temperature;
  const float p_row = a.top_ps ? a.top_ps[row] : a.top_p;
  const float m_row = a.min_ps ? a.min_ps[row] : a.min_p;
  const int k_given = a.top_ks ? a.top_ks[row] : a.top_k;
  const bool greedy = !(t_row > 0.0f);
  const int k_row = greedy ? 1 : k_given;
  const double inv_t = greedy ? 1.0 : 1.0 / (double)t_row;
  const float uu = a.u[row];
  const double u = uu > 0.0f ? (double)fminf(uu, 1.0f) : 0.0;

  auto key_at = [&](int i) { return sample_key(to_f32(x[i])); };
  auto count_above = [&](unsigned k) {  // ids whose key is higher
    int n = 0;
    for (int i = tid; i < V; i += kSampleThreads) n += key_at(i) > k;
    return block_sum(n, iscratch);
  };

  unsigned top = 0;
  for (int i = tid; i < V; i += kSampleThreads) top = max(top, key_at(i));
  top = (unsigned)block_max((double)top, dscratch);
  if (top <= kKeyNegInf) {  // no candidate
    if (tid == 0) a.token[row] = -1;
    if (a.probs)
      for (int i = tid; i < V; i += kSampleThreads) a.probs[row * a.probs_stride + i] = 0.0f;
    return;
  }
  auto mass_above = [&](unsigned k, Cut within) {  // weight of ids whose key is higher than both
    double m = 0.0;
    for (int i = tid; i < V; i += kSampleThreads) {
      const unsigned key = key_at(i);
      if (key > k && key > within.key) m += sample_weight(key, top, inv_t);
    }
    return block_sum(m, dscratch);
  };

  // top-k: the highest key that fewer than k ids are above of, less one, bounds it
  Cut cut{kKeyNegInf, 0};  // every id of weight
  if (k_row > 0 && k_row < V) {
    unsigned lo = kKeyNegInf, hi = top;  // count_above(hi) < k; the answer is in [lo, hi]
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2;
      if (count_above(mid) < k_row) hi = mid;
      else lo = mid + 1;
    }
    cut = Cut{lo, k_row - count_above(lo)};
    if (lo <= kKeyNegInf) cut = Cut{kKeyNegInf, 0};
  }
  const Cut first_k = cut;
  if (!greedy && p_row < 1.0f) {
    const double w_cut = sample_weight(first_k.key, top, inv_t);
    const double total = mass_above(kKeyNegInf, first_k) + first_k.ties * (first_k.key > kKeyNegInf ? w_cut : 0.0);
    const double want = fmax((double)p_row, 0.0) * total;
    unsigned lo = first_k.key, hi = top;  // the least key whose mass above is short of `want`
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2;
      if (mass_above(mid, first_k) < want) hi = mid;
      else lo = mid + 1;
    }
    if (lo > kKeyNegInf) {
      // of the ids with that key, those before which the mass is short of it
      const double above = mass_above(lo, first_k), w = sample_weight(lo, top, inv_t);
      const double more = ceil((want - above) / w);
      cut = shorter(cut, Cut{lo, (int)fmin(fmax(more, 1.0), 2147483647.0)});
    }
  }
  if (!greedy && m_row > 0.0f) {
    unsigned lo = kKeyNegInf + 1, hi = top;  // the least key of weight min_p
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2;
      if (sample_weight(mid, top, inv_t) >= (double)m_row) hi = mid;
      else lo = mid + 1;
    }
    cut = shorter(cut, Cut{lo, 2147483647});
  }

  // ties before an id are counted in the order of ids: threads own whole ranges
  const int per = (V + kSampleThreads - 1) / kSampleThreads;
  const int i0 = min(V, tid * per), i1 = min(V, i0 + per);
  int same = 0, all_same;
  for (int i = i0; i < i1; ++i) same += key_at(i) == cut.key;
  const int before = block_exclusive_scan(same, iscratch, &all_same);
  auto walk = [&](auto &&each) {  // each(id, weight) over this thread's ids
    int tie = before;
    for (int i = i0; i < i1; ++i) {
      const unsigned key = key_at(i);
      const bool kept = key > cut.key || (key == cut.key && tie < cut.ties);
      tie += key == cut.key;
      each(i, kept ? sample_weight(key, top, inv_t) : 0.0);
    }
  };
  double mine = 0.0, total;
  int last = -1;
  walk([&](int i, double w) {
    mine += w;
    if (w > 0.0) last = i;
  });
  if (tid == 0) found = V;
  double run = block_exclusive_scan(mine, dscratch, &total);
  last = (int)block_max((double)last, dscratch);
  const double want = u * total;
  const double inv_total = 1.0 / total;
  int hit = V;
  walk([&](int i, double w) {
    run += w;
    if (w > 0.0 && run > want) hit = min(hit, i);
    if (a.probs) a.probs[row * a.probs_stride + i] = (float)(w * inv_total);
  });
  if (hit < V) atomicMin(&found, hit);
  __syncthreads();
  if (tid == 0) a.token[row] = found < V ? found : last;
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
  const dim3 grid((unsigned)rows), block(kSampleThreads);
  if (dtype == SPECDEC_F32) sample_kernel<float><<<grid, block, 0, as_stream(stream)>>>(a);
  else sample_kernel<__hip_bfloat16><<<grid, block, 0, as_stream(stream)>>>(a);
  return launch_status();
}
