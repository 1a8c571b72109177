// A round's work on a tree of drafted tokens: the attention of its nodes over
// the paged cache and over one another, and the commit of the accepted path.
//
// A tree's nodes are numbered parents first, node 0 the last token of the
// context, which the cache does not hold yet.  Node j of a row that has `past`
// cached positions stands at position past + depth[j].  The nodes' keys and
// values never enter the cache while they are speculative: the attention reads
// them from the projections' rows (rotating k on the way), and the commit, which
// knows the path, appends that path's and nothing else, so a rejected node takes
// no slot and nothing is moved or rolled back.
#include "common.h"

#include <math.h>

namespace specdec {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int kTreeMaxNodes = 256;

struct TreeArgs {
  const void *qkv;  // [batch, nodes, (H + 2 Hkv) d]
  int64_t batch_stride, token_stride;
  const float *cos_t, *sin_t;  // [positions, d / 2]
  int positions;
  const void *k_pool, *v_pool;  // [num_blocks, Hkv, bs, d], [num_blocks, Hkv, d, bs]
  int num_blocks;
  const int32_t *tables;
  int64_t table_stride;
  int table_rows, table_cols;
  const int32_t *meta;
  const int64_t *mask;  // [batch or 1, nodes - first, words]
  int64_t mask_batch_stride, mask_row_stride;
  const int32_t *depth;  // [batch or 1, nodes]
  int64_t depth_batch_stride;
  int batch, nodes, first, H, Hkv, bs;
  float scale;
  void *out;  // [batch, nodes - first, H d]
  int64_t out_batch_stride, out_token_stride;
};

// A row's metadata; `fits` is false where they reach outside the tables.
struct TreeRow {
  int row, past, live;
  bool fits;
};
__device__ __forceinline__ TreeRow tree_row(const TreeArgs &a, int b) {
  TreeRow r{a.meta[b], a.meta[a.batch + b], a.meta[2 * a.batch + b], true};
  r.live = min(r.live, a.nodes);
  r.fits = r.row >= 0 && r.row < a.table_rows && r.past >= 0 && r.past <= (int64_t)a.table_cols * a.bs;
  return r;
}

// One wave a (query node, head): a lane a key, 64 keys at a time, in fp32.  For
// what the tiles below do not take: blocks that are no multiple of 16 bytes of
// keys, rows that are not 16-byte aligned.  Bound by its scattered reads (8 rows of
// 32 nodes at 4096 keys, 32 heads: 4.1 ms).
template <typename T, int D>
__global__ __launch_bounds__(kWave) void tree_attention_any_kernel(TreeArgs a) {
  const int lane = threadIdx.x, b = blockIdx.z, h = blockIdx.y, i = blockIdx.x, node = a.first + i;
  const TreeRow r = tree_row(a, b);
  if (node >= r.live) return;
  const int hk = h / (a.H / a.Hkv);
  const T *rows = (const T *)a.qkv + b * a.batch_stride;
  T *out = (T *)a.out + b * a.out_batch_stride + i * a.out_token_stride + h * D;
  const int32_t *depth = a.depth + b * a.depth_batch_stride;
  const int64_t *mask = a.mask + b * a.mask_batch_stride + i * a.mask_row_stride;
  constexpr int HALF = D / 2, PER = D / kWave;
  __shared__ float q[D];
  // cos and sin of a position, NaN outside the tables
  auto angle = [&](int pos, int j, float &c, float &s) {
    const bool in = pos >= 0 && pos < a.positions;
    c = in ? a.cos_t[(int64_t)pos * HALF + j] : NAN;
    s = in ? a.sin_t[(int64_t)pos * HALF + j] : NAN;
  };
  if (lane < HALF) {
    const T *src = rows + node * a.token_stride + h * D;
    float c, s, y1, y2;
    angle(r.past + depth[node], lane, c, s);
    rope_pair(to_f32(src[lane]), to_f32(src[lane + HALF]), c, s, y1, y2);
    q[lane] = to_f32(from_f32<T>(y1));
    q[lane + HALF] = to_f32(from_f32<T>(y2));
  }
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o[PER] = {};
  bool good = r.fits;
  // a step of 64 keys: this lane's score, and the value row of any key of the step
  auto step = [&](float score, auto &&value) {
    if (!__any(score != -INFINITY)) return;  // a NaN is seen, and passes the maximum by
    const float m_new = fmaxf(m, wave_max(score));
    const float p = score == -INFINITY ? 0.0f : expf(score - m_new);
    const float keep = m == -INFINITY ? 0.0f : expf(m - m_new);
    m = m_new;
    l = l * keep + wave_sum(p);
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] *= keep;
    for (int j = 0; j < kWave; ++j) {
      const float pj = __shfl(p, j, kWave);
      if (pj == 0.0f) continue;
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] += pj * value(j, lane + e * kWave);
    }
  };
  const int past = r.fits ? r.past : 0;
  const int32_t *table = a.tables + (r.fits ? r.row * a.table_stride : 0);
  for (int k0 = 0; k0 < past; k0 += kWave) {
    const int key = k0 + lane;
    int id = key < past ? table[key / a.bs] : 0;
    if (id < 0 || id >= a.num_blocks) {
      id = 0;
      good = false;
    }
    const int64_t at = ((int64_t)id * a.Hkv + hk) * a.bs * D;
    float score = -INFINITY;
    if (key < past) {
      const T *k = (const T *)a.k_pool + at + (int64_t)(key % a.bs) * D;
      float dot = 0.0f;
      for (int j = 0; j < D; ++j) dot += q[j] * to_f32(k[j]);
      score = dot * a.scale;
    }
    step(score, [&](int j, int dim) {
      const int64_t tile = __shfl(at, j, kWave);
      return to_f32(((const T *)a.v_pool)[tile + (int64_t)dim * a.bs + (k0 + j) % a.bs]);
    });
  }
  for (int k0 = 0; k0 < r.live; k0 += kWave) {
    const int key = k0 + lane;
    float score = -INFINITY;
    if (key < r.live && (mask[k0 / kWave] >> lane & 1)) {
      const T *k = rows + key * a.token_stride + (a.H + hk) * D;
      float dot = 0.0f;
      for (int j = 0; j < HALF; ++j) {
        float c, s, y1, y2;
        angle(r.past + depth[key], j, c, s);
        rope_pair(to_f32(k[j]), to_f32(k[j + HALF]), c, s, y1, y2);
        dot += q[j] * to_f32(from_f32<T>(y1)) + q[j + HALF] * to_f32(from_f32<T>(y2));
      }
      score = dot * a.scale;
    }
    step(score, [&](int j, int dim) {
      return to_f32(rows[(k0 + j) * a.token_stride + (a.H + a.Hkv + hk) * D + dim]);
    });
  }
  good = __all(good);
#pragma unroll
  for (int e = 0; e < PER; ++e)
    out[lane + e * kWave] = from_f32<T>(!good ? NAN : l > 0.0f || l != l ? o[e] / l : 0.0f);
}

// The grid of matrix-instruction tiles.
//
// A wave owns chunks of CK keys (32 in bf16, 16 in fp32: 4 lane groups of a
// 16-byte piece) and up to NT tiles of 16 query rows, the nodes and query heads
// of one kv head.  With lane = 16 g + c:
//   S^T[key, query] = K Q^T    A: K row of lane c, B: query c, pieces of 16 bytes
//                              at dims CK j + EPL g
//   O^T[dim, query] += V^T P^T A: V row of dim 16 t + c, keys EPL g .. + EPL - 1
// Row 4 g + i of score tile t is key EPL g + 4 t + i of the chunk, so the scores
// that a lane holds are the keys of the V piece that it loads: P goes from one
// product to the next in registers, and K and V pass from memory to registers
// once for all of the wave's query rows, with no LDS and no barrier before the
// end, where the workgroup's waves fold their (m, l, O).
// A lane's row of K holds pieces j and j + NP / 2 of a rotated pair of dims, so the
// tree's own keys are rotated in the registers that they arrive in.
// In bf16 the second product takes P in bf16, as the other attention kernels here do:
// each weight is off by 2^-8 of itself at most, while l sums them in fp32 as they
// were.  Two halves of P would double that product's instructions.  Against 64 bits the
// outputs are off by 0.0021 to 0.0022 of their size where one rounding at the end
// leaves 0.0016 to 0.0017 (the bf16 cases of perf/more_operators.py).
// Bound by memory: 8 rows of 32 nodes at 4096 keys, 32 heads of 64, 55 us for 241 MB
// (85% of a copy's rate); by the dependent round trips of metadata, tables, nodes
// and keys where these are few (one row of 16 nodes at 300 keys 7.3 us).
constexpr int kTreeWaves = 4;

template <typename T, int D> struct TreeTile {
  static constexpr int EPL = 16 / sizeof(T);  // elements of a piece
  static constexpr int CK = 4 * EPL;
  static constexpr int NTK = CK / 16;  // score tiles of a chunk
  static constexpr int NP = D / CK;    // pieces of a lane's K or Q row
  static constexpr int ND = D / 16;    // pieces of V, tiles of O
};

__device__ __forceinline__ f32x4 tree_mma(__hip_bfloat16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 tree_mma(float, u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ void tree_unpack(u32x4 v, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __uint_as_float((e & 1) ? v[e / 2] & 0xFFFF0000u : v[e / 2] << 16);
}
__device__ __forceinline__ void tree_unpack(u32x4 v, float (&x)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[e]);
}
__device__ __forceinline__ u32x4 tree_pack(const float (&x)[8]) {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (__bf16)x[e];  // to nearest even
  return __builtin_bit_cast(u32x4, v);
}
__device__ __forceinline__ u32x4 tree_pack(const float (&x)[4]) {
  return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
}

// The pieces lo = dims d .. d + EPL - 1 and hi = those half a head later, rotated at a position.
template <int EPL> __device__ __forceinline__ void tree_rotate(u32x4 &lo, u32x4 &hi, const float *c, const float *s, bool in) {
  float x1[EPL], x2[EPL];
  tree_unpack(lo, x1);
  tree_unpack(hi, x2);
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    float y1, y2;
    rope_pair(x1[e], x2[e], in ? c[e] : NAN, in ? s[e] : NAN, y1, y2);
    x1[e] = y1;
    x2[e] = y2;
  }
  lo = tree_pack(x1);
  hi = tree_pack(x2);
}

// Row pieces of a q or k row at a position of the tree, rotated and rounded.
template <typename T, int D>
__device__ __forceinline__ void tree_row_pieces(const TreeArgs &a, const T *row, int64_t pos, int g,
                                                u32x4 (&r)[TreeTile<T, D>::NP]) {
  using L = TreeTile<T, D>;
  const bool in = pos >= 0 && pos < a.positions;
  const int64_t at = in ? pos * (D / 2) : 0;
#pragma unroll
  for (int j = 0; j < L::NP; ++j) r[j] = *(const u32x4 *)(row + L::CK * j + L::EPL * g);
#pragma unroll
  for (int j = 0; j < L::NP / 2; ++j) {
    float c[L::EPL], s[L::EPL];
#pragma unroll
    for (int e = 0; e < L::EPL; e += 4) {
      *(f32x4 *)&c[e] = *(const f32x4 *)(a.cos_t + at + L::CK * j + L::EPL * g + e);
      *(f32x4 *)&s[e] = *(const f32x4 *)(a.sin_t + at + L::CK * j + L::EPL * g + e);
    }
    tree_rotate<L::EPL>(r[j], r[j + L::NP / 2], c, s, in);
  }
}

// The scale of scores in log2 units, above 0 so that a hidden key's -inf stays that
// and the largest score is the largest after it: a negative scale is taken into q's
// sign (exact), and 0 is the least fp32 number, which leaves every finite score less
// than 2^-20.
__device__ __forceinline__ float tree_scale(float scale) {
  const float sc = fabsf(scale) * 1.4426950408889634f;
  return sc == 0.0f ? 0x1p-149f : sc;
}
template <typename T> __device__ __forceinline__ unsigned tree_sign(float scale) {
  return scale < 0.0f ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
}

// How a call is cut: tiles of a wave, groups of them over a kv head's query
// rows, splits over the cached keys.
struct TreeCut {
  int tiles, groups, splits;
  bool shared;  // the grid whose waves share their keys
  __host__ __device__ int64_t rows() const { return (int64_t)groups * tiles * 16; }  // of a kv head, with padding
};

// Split partials: for each (row, kv head, split) the query rows' m and l, then
// their O, not divided.
struct TreeParts {
  float *ml, *o;
};
__host__ __device__ inline TreeParts tree_parts(float *ws, int64_t unit, int64_t units, int64_t rows, int d) {
  return TreeParts{ws + unit * rows * 2, ws + units * rows * 2 + unit * rows * d};
}

// Waves a SIMD that a variant's registers are held to: 168, 256 and 512 of them
// for q, O, two chunks of K and V and the tree's tables.
constexpr int tree_waves(int d, int tiles) { return (d == 64 ? 4 : 3) - tiles; }

template <typename T, int D, int NT>
__global__ __launch_bounds__(kTreeWaves *kWave)
    __attribute__((amdgpu_waves_per_eu(tree_waves(D, NT), tree_waves(D, NT)))) void tree_attention_kernel(TreeArgs a, TreeCut cut, int shift, float *ws) {
  using L = TreeTile<T, D>;
  constexpr int EPL = L::EPL, CK = L::CK, NTK = L::NTK, NP = L::NP, ND = L::ND, NW = kTreeWaves;
  constexpr int MT = NT < 2 ? 1 : 2;  // tiles folded at a time
  __shared__ float s_o[NW][MT][16][D + 4];
  __shared__ float s_ml[NW][MT][16][2];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, c = lane & 15, g = lane / 16;
  const int units = a.batch * a.Hkv * cut.splits, unit = blockIdx.x;
  const int split = unit % cut.splits, bh = unit / cut.splits, hk = bh % a.Hkv, b = bh / a.Hkv;
  const int G = a.H / a.Hkv;
  const TreeRow r = tree_row(a, b);
  const int nrows = (r.live - a.first) * G;
  if (nrows <= 0) return;
  const int tiles = min(NT, (nrows + 15) / 16);
  bool bad = !r.fits;
  const int past = r.fits ? r.past : 0, live = r.live;
  const T *rows = (const T *)a.qkv + b * a.batch_stride;
  const int32_t *depth = a.depth + b * a.depth_batch_stride;
  const int32_t *table = a.tables + (r.fits ? r.row * a.table_stride : 0);

  u32x4 q[NT][NP];
  f32x4 o[NT][ND];
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int qr = min(16 * t + c, nrows - 1), node = a.first + qr / G;
    if (t < tiles) {
      tree_row_pieces<T, D>(a, rows + node * a.token_stride + (int64_t)(hk * G + qr % G) * D, (int64_t)r.past + depth[node], g,
                            q[t]);
#pragma unroll
      for (int j = 0; j < NP; ++j) q[t][j] ^= tree_sign<T>(a.scale);
    }
    m[t] = -INFINITY;
    l[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float sc = tree_scale(a.scale);

  // the chunk's weights of tile t, in log2 units against the running maximum,
  // which is raised when a score passes it by 2^8 only: rarely after the first
  // chunks, and p <= 2^8 loses nothing
  auto weigh = [&](int t, float (&s)[EPL]) {
    float top = s[0];
#pragma unroll
    for (int e = 1; e < EPL; ++e) top = fmaxf(top, s[e]);
    top *= sc;
    if (__any(top > m[t] + 8.0f)) {
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float m_new = fmaxf(m[t], top);
      const float f = m[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[t] - m_new);
      m[t] = m_new;
      l[t] *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[t][d] *= f;
    }
    const float base = m[t] == -INFINITY ? 0.0f : m[t];
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], sc, -base));
      l[t] += s[e];
    }
  };
  auto scores = [&](int t, const u32x4 (&k)[NTK][NP], float (&s)[EPL]) {
#pragma unroll
    for (int tk = 0; tk < NTK; ++tk) {
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NP; ++j) acc = tree_mma(T(), k[tk][j], q[t][j], acc);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * tk + i] = acc[i];
    }
  };

  // ---- the tree's own keys, chunks dealt over the splits' waves
  for (int n0 = (wave * cut.splits + split) * CK; n0 < live; n0 += NW * cut.splits * CK) {
    u32x4 k[NTK][NP], v[ND];
#pragma unroll
    for (int tk = 0; tk < NTK; ++tk) {
      const int node = min(n0 + EPL * (c / 4) + 4 * tk + c % 4, live - 1);
      tree_row_pieces<T, D>(a, rows + node * a.token_stride + (int64_t)(a.H + hk) * D, (int64_t)r.past + depth[node], g, k[tk]);
    }
    // V rows are tokens here: a piece's keys are gathered
    const T *vrows = rows + (int64_t)(a.H + a.Hkv + hk) * D;
    bool finite = true;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      float x[EPL];
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        x[e] = to_f32(vrows[min(n0 + EPL * g + e, live - 1) * a.token_stride + 16 * d + c]);
        finite &= fabsf(x[e]) < INFINITY;
      }
      v[d] = tree_pack(x);
    }
    finite = __all(finite);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t >= tiles) break;
      float s[EPL];
      scores(t, k, s);
      const int qr = min(16 * t + c, nrows - 1);
      const uint64_t word = a.mask[b * a.mask_batch_stride + qr / G * a.mask_row_stride + n0 / 64];
      const unsigned seen = (unsigned)(word >> (n0 % 64 + EPL * g));
#pragma unroll
      for (int e = 0; e < EPL; ++e)
        if (!(seen >> e & 1) || n0 + EPL * g + e >= live) s[e] = -INFINITY;
      weigh(t, s);
      if (finite) {
        const u32x4 p = tree_pack(s);
#pragma unroll
        for (int d = 0; d < ND; ++d) o[t][d] = tree_mma(T(), v[d], p, o[t][d]);
      } else {
        // a value that is no number reaches the queries that see its node, and
        // no other: 0 times it is left out, key by key
        for (int key = 0; key < min(CK, live - n0); ++key) {
          float pk = 0.0f;
#pragma unroll
          for (int e = 0; e < EPL; ++e) pk = key % EPL == e ? s[e] : pk;
          pk = __shfl(pk, key / EPL * 16 + c, kWave);
          if (pk == 0.0f) continue;
          const T *vr = vrows + (n0 + key) * a.token_stride + 4 * g;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][d][i] += pk * to_f32(vr[16 * d + i]);
        }
      }
    }
  }

  // ---- the cached keys: this split's chunks, dealt over its waves
  const int chunks = (past + CK - 1) / CK, per = (chunks + cut.splits - 1) / cut.splits;
  const int end = min(chunks, (split + 1) * per);
  const int64_t tile = (int64_t)a.bs * D, stride = tile * a.Hkv;
  const T *kp = (const T *)a.k_pool + hk * tile, *vp = (const T *)a.v_pool + hk * tile;
  const int last_run = (past - 1) & ~(EPL - 1);
  struct Where {
    int k_id, v_id, k_slot, v_slot;
  };
  auto block_of = [&](int key, int &slot) {
    const int j = shift >= 0 ? key >> shift : key / a.bs;
    slot = key - j * a.bs;
    return table[j];
  };
  auto where = [&](int ch) {
    Where w;
    w.k_id = block_of(min(ch * CK + EPL * (c / 4), last_run), w.k_slot);
    w.v_id = block_of(min(ch * CK + EPL * g, last_run), w.v_slot);
    return w;
  };
  struct Pieces {
    u32x4 k[NTK][NP], v[ND];
  };
  auto load = [&](const Where &w, Pieces &x) {
    bad |= (unsigned)w.k_id >= (unsigned)a.num_blocks || (unsigned)w.v_id >= (unsigned)a.num_blocks;
    const unsigned most = a.num_blocks - 1;
    const T *k = kp + min((unsigned)w.k_id, most) * stride + (int64_t)(w.k_slot + c % 4) * D + EPL * g;
    const T *v = vp + min((unsigned)w.v_id, most) * stride + (int64_t)c * a.bs + w.v_slot;
#pragma unroll
    for (int tk = 0; tk < NTK; ++tk)
#pragma unroll
      for (int j = 0; j < NP; ++j) x.k[tk][j] = *(const u32x4 *)(k + 4 * tk * D + CK * j);
#pragma unroll
    for (int d = 0; d < ND; ++d) x.v[d] = *(const u32x4 *)(v + (int64_t)16 * d * a.bs);
  };
  auto compute = [&](int ch, Pieces &x) {
    const int left = past - ch * CK - EPL * g;  // keys of this lane's V piece that there are, or more
    const bool edge = (ch + 1) * CK > past;
    if (edge) {  // slots behind the cached length hold anything at all
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (sizeof(T) == 2)
            x.v[d][w] = 2 * w + 1 < left ? x.v[d][w] : 2 * w < left ? x.v[d][w] & 0xFFFFu : 0u;
          else
            x.v[d][w] = w < left ? x.v[d][w] : 0u;
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t >= tiles) break;
      float s[EPL];
      scores(t, x.k, s);
      if (edge) {
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          if (e >= left) s[e] = -INFINITY;
      }
      weigh(t, s);
      const u32x4 p = tree_pack(s);
#pragma unroll
      for (int d = 0; d < ND; ++d) o[t][d] = tree_mma(T(), x.v[d], p, o[t][d]);
    }
  };
  int ch = split * per + wave;
  if (ch < end) {
    // block ids two chunks ahead of the products, K and V one
    Pieces x0, x1;
    load(where(ch), x0);
    Where w = where(min(ch + NW, end - 1));
    while (true) {
      if (ch + NW >= end) {
        compute(ch, x0);
        break;
      }
      load(w, x1);
      w = where(min(ch + 2 * NW, end - 1));
      compute(ch, x0);
      ch += NW;
      if (ch + NW >= end) {
        compute(ch, x1);
        break;
      }
      load(w, x0);
      w = where(min(ch + 2 * NW, end - 1));
      compute(ch, x1);
      ch += NW;
    }
  }

  // ---- fold the waves, MT tiles at a time
  bad = __any(bad);
  const TreeParts parts = tree_parts(ws, unit, units, cut.rows(), D);
#pragma unroll
  for (int t0 = 0; t0 < NT; t0 += MT) {
    if (t0 >= tiles) break;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      const int t = t0 + u;
      float sum = l[t] + __shfl_xor(l[t], 16, kWave);
      sum += __shfl_xor(sum, 32, kWave);
      if (g == 0) {
        s_ml[wave][u][c][0] = m[t];
        s_ml[wave][u][c][1] = bad ? NAN : sum;
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) *(f32x4 *)&s_o[wave][u][c][16 * d + 4 * g] = o[t][d];
    }
    __syncthreads();
    for (int x = tid; x < MT * 16 * (D / 4); x += NW * kWave) {
      const int u = x / (4 * D), rr = x / (D / 4) % 16, d = x % (D / 4) * 4;
      const int qr = 16 * (t0 + u) + rr;
      if (qr >= nrows) continue;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) top = fmaxf(top, s_ml[w][u][rr][0]);
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = s_ml[w][u][rr][0], f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - top);
        const float lw = s_ml[w][u][rr][1];
        sum += mw == -INFINITY ? lw : lw * f;  // 0, or NaN
        acc += f * *(const f32x4 *)&s_o[w][u][rr][d];
      }
      if (cut.splits > 1) {
        *(f32x4 *)&parts.o[(int64_t)qr * D + d] = acc;
        if (d == 0) {
          parts.ml[qr * 2] = top;
          parts.ml[qr * 2 + 1] = sum;
        }
      } else {
        T *out = (T *)a.out + b * a.out_batch_stride + qr / G * a.out_token_stride + (int64_t)(hk * G + qr % G) * D + d;
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = from_f32<T>(sum != 0.0f ? acc[i] * inv : 0.0f);
      }
    }
  }
}

// The same for more than 32 query rows a kv head: NW waves share a chunk of 2 CK
// keys through LDS, each with up to NT tiles of its own, so the keys are read once
// for 16 NT NW query rows and no wave's state has to be folded with another's.
// The next chunk is in flight in registers while this one is used; one barrier a
// chunk, two buffers.  Against the grid above with four tiles a wave: 8 rows of 64
// nodes at 4096 keys, one query head a kv head, 85 -> 65 us (73% of the bytes at a
// copy's rate); 4 rows of 64 nodes at 8000 keys, four query heads a kv head of 64,
// 72 -> 46, and of 128, where that grid has room for two tiles, 116 -> 76.  There it
// is bound by its instructions: 11.6 k vector and 1.8 k matrix instructions a SIMD
// are some 31 of the 63 us, with two waves a SIMD to hide the rest; the splits'
// partials (34 MB) and their fold are most of the others.
// K is kept in the order of the score tiles' rows, rows of 4 NP pieces; V as in the
// cache, rows of 8 pieces; a piece's place in its row is its number xor the row's
// low bits, so that the lanes of a read fall on different banks.
template <typename T, int D, int NW> struct TreeShared {
  using L = TreeTile<T, D>;
  static constexpr int KC = 2 * L::CK, PR = 4 * L::NP, THREADS = NW * kWave;
  static constexpr int KS = KC * PR / THREADS, VS = D * 8 / THREADS;  // pieces that a thread brings
  static_assert(KS > 0 && VS > 0 && KS * THREADS == KC * PR && VS * THREADS == D * 8, "whole pieces a thread");
  u32x4 k[2][KC * PR], v[2][D * 8];
  int odd;  // a value of the tree is no number
  static __device__ __forceinline__ int k_at(int key, int p) {  // of a chunk's key, piece p of its row
    const int in = key % L::CK, row = (key / L::CK * L::NTK + in % L::EPL / 4) * 16 + in / L::EPL * 4 + in % 4;
    return row * PR + (p ^ (row & 7));
  }
  static __device__ __forceinline__ int v_at(int d, int p) { return d * 8 + (p ^ (d & 7)); }
};

template <typename T, int D, int NW, int NT>
__global__ __launch_bounds__(NW *kWave) __attribute__((amdgpu_waves_per_eu(NT == 1 ? 4 : 2, NT == 1 ? 4 : 2))) void
tree_attention_shared_kernel(TreeArgs a, TreeCut cut, int shift, float *ws) {
  using L = TreeTile<T, D>;
  using S = TreeShared<T, D, NW>;
  constexpr int EPL = L::EPL, CK = L::CK, NTK = L::NTK, NP = L::NP, ND = L::ND, KC = S::KC, PR = S::PR;
  __shared__ S sh;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, c = lane & 15, g = lane / 16;
  const int units = a.batch * a.Hkv * cut.splits;
  // query groups that read the same keys run next to one another on one XCD,
  // whose L2 then serves all but the first (workgroups go to the XCDs in turn)
  int unit = blockIdx.x, qg = 0;
  if (cut.groups > 1) {
    const int rest = unit / 8;
    qg = rest % cut.groups;
    unit = rest / cut.groups * 8 + unit % 8;
    if (unit >= units) return;
  }
  const int split = unit % cut.splits, bh = unit / cut.splits, hk = bh % a.Hkv, b = bh / a.Hkv;
  const int G = a.H / a.Hkv;
  const TreeRow r = tree_row(a, b);
  const int row0 = qg * cut.tiles * 16, nrows = (r.live - a.first) * G;
  if (row0 >= nrows) return;
  bool bad = !r.fits;
  const int past = r.fits ? r.past : 0, live = r.live;
  const T *rows = (const T *)a.qkv + b * a.batch_stride;
  const int32_t *depth = a.depth + b * a.depth_batch_stride;
  const int32_t *table = a.tables + (r.fits ? r.row * a.table_stride : 0);
  const auto first_row = [&](int t) { return row0 + 16 * (wave + NW * t); };  // of this wave's tile t
  int tiles = 0;

  u32x4 q[NT][NP];
  f32x4 o[NT][ND];
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (first_row(t) < nrows) tiles = t + 1;
    const int qr = min(first_row(t) + c, nrows - 1), node = a.first + qr / G;
    tree_row_pieces<T, D>(a, rows + node * a.token_stride + (int64_t)(hk * G + qr % G) * D, (int64_t)r.past + depth[node], g,
                          q[t]);
#pragma unroll
    for (int j = 0; j < NP; ++j) q[t][j] ^= tree_sign<T>(a.scale);
    m[t] = -INFINITY;
    l[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float sc = tree_scale(a.scale);

  // half a chunk (CK keys) of buffer `buf` against this wave's tiles; hide(t, s) puts
  // the scores of keys that a query does not see to -inf
  const auto use = [&](int buf, int half, bool odd, int keys, auto &&hide) __attribute__((always_inline)) {
    if (tiles == 0) return;
    float s[NT][EPL];
#pragma unroll
    for (int tk = 0; tk < NTK; ++tk) {
      const int row = (half * NTK + tk) * 16 + c;
      u32x4 k[NP];
#pragma unroll
      for (int j = 0; j < NP; ++j) k[j] = sh.k[buf][row * PR + ((4 * j + g) ^ (row & 7))];
      f32x4 acc[NT];  // a tile that the wave does not have costs less than the branches around it
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NP; ++j)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = tree_mma(T(), k[j], q[t][j], acc[t]);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][4 * tk + i] = acc[t][i];
    }
    // K's registers are free before V's are taken: all at once are spilled, and a
    // reload waits for the chunk in flight
    __builtin_amdgcn_sched_barrier(0);
    constexpr int VN = ND < 4 ? ND : 4;
    u32x4 v[VN], p[NT];
    const auto take = [&](int d0) __attribute__((always_inline)) {
#pragma unroll
      for (int d = 0; d < VN; ++d) v[d] = sh.v[buf][S::v_at(16 * (d0 + d) + c, half * 4 + g)];
    };
    take(0);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      hide(t, s[t]);
      float top = s[t][0];
#pragma unroll
      for (int e = 1; e < EPL; ++e) top = fmaxf(top, s[t][e]);
      top *= sc;
      if (__any(top > m[t] + 8.0f)) {  // as above
        top = fmaxf(top, __shfl_xor(top, 16, kWave));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const float m_new = fmaxf(m[t], top);
        const float f = m[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[t] - m_new);
        m[t] = m_new;
        l[t] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[t][d] *= f;
      }
      const float base = m[t] == -INFINITY ? 0.0f : m[t];
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        s[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], sc, -base));
        l[t] += s[t][e];
      }
      p[t] = tree_pack(s[t]);
      if (odd) {
        for (int key = 0; key < keys; ++key) {  // 0 times what is no number is left out
          float pk = 0.0f;
#pragma unroll
          for (int e = 0; e < EPL; ++e) pk = key % EPL == e ? s[t][e] : pk;
          pk = __shfl(pk, key / EPL * 16 + c, kWave);
          if (pk == 0.0f) continue;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              o[t][d][i] += pk * to_f32(((const T *)&sh.v[buf][S::v_at(16 * d + 4 * g + i, half * 4 + key / EPL)])[key % EPL]);
        }
      }
    }
    if (odd) return;
#pragma unroll
    for (int d0 = 0; d0 < ND; d0 += VN) {
      if (d0 > 0) {
        take(d0);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int d = 0; d < VN; ++d)
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][d0 + d] = tree_mma(T(), v[d], p[t], o[t][d0 + d]);
    }
  };

  // ---- the tree's own keys, chunks dealt over the splits
  for (int n0 = split * KC; n0 < live; n0 += cut.splits * KC) {
    __syncthreads();
    if (tid == 0) sh.odd = 0;
    __syncthreads();
    for (int i = tid; i < KC * PR / 2; i += S::THREADS) {
      const int key = i / (PR / 2), p = i % (PR / 2), node = min(n0 + key, live - 1);
      const int64_t pos = (int64_t)r.past + depth[node];
      const bool in = pos >= 0 && pos < a.positions;
      const T *row = rows + node * a.token_stride + (int64_t)(a.H + hk) * D + EPL * p;
      u32x4 lo = *(const u32x4 *)row, hi = *(const u32x4 *)(row + D / 2);
      float co[EPL], si[EPL];
#pragma unroll
      for (int e = 0; e < EPL; e += 4) {
        *(f32x4 *)&co[e] = *(const f32x4 *)(a.cos_t + (in ? pos : 0) * (D / 2) + EPL * p + e);
        *(f32x4 *)&si[e] = *(const f32x4 *)(a.sin_t + (in ? pos : 0) * (D / 2) + EPL * p + e);
      }
      tree_rotate<EPL>(lo, hi, co, si, in);
      sh.k[0][S::k_at(key, p)] = lo;
      sh.k[0][S::k_at(key, p + PR / 2)] = hi;
    }
    for (int i = tid; i < KC * PR; i += S::THREADS) {
      const int key = i / PR, p = i % PR, node = min(n0 + key, live - 1);
      const u32x4 v = *(const u32x4 *)(rows + node * a.token_stride + (int64_t)(a.H + a.Hkv + hk) * D + EPL * p);
      float x[EPL];
      tree_unpack(v, x);
      bool finite = true;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        finite &= fabsf(x[e]) < INFINITY;
        ((T *)&sh.v[0][S::v_at(EPL * p + e, key / EPL)])[key % EPL] = from_f32<T>(x[e]);
      }
      if (!finite) sh.odd = 1;
    }
    __syncthreads();
    const bool odd = sh.odd != 0;
#pragma unroll 1
    for (int half = 0; half < 2; ++half)
      use(0, half, odd, min(CK, max(0, live - n0 - half * CK)), [&](int t, float(&s)[EPL]) __attribute__((always_inline)) {
        const int key = n0 + half * CK + EPL * g, qr = min(first_row(t) + c, nrows - 1);
        const uint64_t word = key < live ? a.mask[b * a.mask_batch_stride + qr / G * a.mask_row_stride + key / 64] : 0;
        const unsigned seen = (unsigned)(word >> (key % 64));
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          if (!(seen >> e & 1) || key + e >= live) s[e] = -INFINITY;
      });
  }

  // ---- the cached keys: this split's chunks
  const int chunks = (past + KC - 1) / KC, per = (chunks + cut.splits - 1) / cut.splits;
  const int begin = split * per, end = min(chunks, begin + per);
  const int64_t tile = (int64_t)a.bs * D, stride = tile * a.Hkv;
  const T *kp = (const T *)a.k_pool + hk * tile, *vp = (const T *)a.v_pool + hk * tile;
  const unsigned most = a.num_blocks - 1;
  struct Ids {
    int k[S::KS], v[S::VS];
  };
  struct Brought {
    u32x4 k[S::KS], v[S::VS];
  };
  const auto page = [&](int key) { return shift >= 0 ? key >> shift : key / a.bs; };
  const auto k_key = [&](int ch, int i) { return min(ch * KC + (tid + i * S::THREADS) / PR, past - 1); };
  const auto v_key = [&](int ch, int i) {
    return min(ch * KC + (tid + i * S::THREADS) % 8 * EPL, (past - 1) & ~(EPL - 1));
  };
  const auto look = [&](int ch, Ids &w) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < S::KS; ++i) w.k[i] = table[page(k_key(ch, i))];
#pragma unroll
    for (int i = 0; i < S::VS; ++i) w.v[i] = table[page(v_key(ch, i))];
  };
  const auto bring = [&](int ch, const Ids &w, Brought &x) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < S::KS; ++i) {
      bad |= (unsigned)w.k[i] > most;
      const int key = k_key(ch, i);
      x.k[i] = *(const u32x4 *)(kp + min((unsigned)w.k[i], most) * stride + (int64_t)(key - page(key) * a.bs) * D +
                                (tid + i * S::THREADS) % PR * EPL);
    }
#pragma unroll
    for (int i = 0; i < S::VS; ++i) {
      bad |= (unsigned)w.v[i] > most;
      const int key = v_key(ch, i);
      x.v[i] = *(const u32x4 *)(vp + min((unsigned)w.v[i], most) * stride + (int64_t)((tid + i * S::THREADS) / 8) * a.bs + key -
                                page(key) * a.bs);
    }
  };
  const auto put = [&](int ch, int buf, Brought &x) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < S::KS; ++i) sh.k[buf][S::k_at((tid + i * S::THREADS) / PR, (tid + i * S::THREADS) % PR)] = x.k[i];
#pragma unroll
    for (int i = 0; i < S::VS; ++i) {
      const int p = (tid + i * S::THREADS) % 8, left = past - ch * KC - p * EPL;
      if (left < EPL) {  // slots behind the cached length hold anything at all
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (sizeof(T) == 2)
            x.v[i][w] = 2 * w + 1 < left ? x.v[i][w] : 2 * w < left ? x.v[i][w] & 0xFFFFu : 0u;
          else
            x.v[i][w] = w < left ? x.v[i][w] : 0u;
        }
      }
      sh.v[buf][S::v_at((tid + i * S::THREADS) / 8, p)] = x.v[i];
    }
  };
  if (begin < end) {
    Ids w;
    Brought x;
    look(begin, w);
    bring(begin, w, x);
    look(min(begin + 1, end - 1), w);
    __syncthreads();  // the tree's chunk has been used
    put(begin, 0, x);
    __syncthreads();
    for (int ch = begin; ch < end; ++ch) {
      const int buf = (ch - begin) & 1;
      if (ch + 1 < end) {
        bring(ch + 1, w, x);
        look(min(ch + 2, end - 1), w);
      }
#pragma unroll 1
      for (int half = 0; half < 2; ++half)
        use(buf, half, false, 0, [&](int, float(&s)[EPL]) __attribute__((always_inline)) {
          const int left = past - ch * KC - half * CK - EPL * g;
          if (left < EPL) {
#pragma unroll
            for (int e = 0; e < EPL; ++e)
              if (e >= left) s[e] = -INFINITY;
          }
        });
      if (ch + 1 < end) put(ch + 1, buf ^ 1, x);
      __syncthreads();
    }
  }
  bad = __syncthreads_or(bad);

  const TreeParts parts = tree_parts(ws, unit, units, cut.rows(), D);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t >= tiles) break;
    float sum = l[t] + __shfl_xor(l[t], 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    if (bad) sum = NAN;
    const int qr = first_row(t) + c;
    if (qr >= nrows) continue;
    if (cut.splits > 1) {
      if (g == 0) {
        parts.ml[qr * 2] = m[t];
        parts.ml[qr * 2 + 1] = sum;
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) *(f32x4 *)&parts.o[(int64_t)qr * D + 16 * d + 4 * g] = o[t][d];
    } else {
      T *out = (T *)a.out + b * a.out_batch_stride + qr / G * a.out_token_stride + (int64_t)(hk * G + qr % G) * D + 4 * g;
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) out[16 * d + i] = from_f32<T>(sum != 0.0f ? o[t][d][i] * inv : 0.0f);
    }
  }
}

// Folds the splits' partials, D / 4 lanes a query row.
template <typename T, int D> __global__ __launch_bounds__(256) void tree_fold_kernel(TreeArgs a, TreeCut cut, float *ws) {
  constexpr int LANES = D / 4, PER = 256 / LANES;
  const int b = blockIdx.z, hk = blockIdx.y, G = a.H / a.Hkv, S = cut.splits;
  const int qr = blockIdx.x * PER + threadIdx.x / LANES, d = threadIdx.x % LANES * 4;
  const int live = min(a.meta[2 * a.batch + b], a.nodes);
  if (qr >= (live - a.first) * G) return;
  const int64_t units = (int64_t)a.batch * a.Hkv * S, unit0 = ((int64_t)b * a.Hkv + hk) * S, rows = cut.rows();
  float top = -INFINITY, sum = 0.0f;
  for (int s = 0; s < S; ++s) top = fmaxf(top, tree_parts(ws, unit0 + s, units, rows, D).ml[qr * 2]);
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < S; ++s) {
    const TreeParts p = tree_parts(ws, unit0 + s, units, rows, D);
    const float ms = p.ml[qr * 2], ls = p.ml[qr * 2 + 1];
    const float f = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - top);
    sum += ms == -INFINITY ? ls : ls * f;
    acc += f * *(const f32x4 *)&p.o[(int64_t)qr * D + d];
  }
  T *out = (T *)a.out + b * a.out_batch_stride + qr / G * a.out_token_stride + (int64_t)(hk * G + qr % G) * D + d;
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = from_f32<T>(sum != 0.0f ? acc[i] * inv : 0.0f);
}

// Cut of a call whose rows hold up to max_kv cached keys.
inline TreeCut tree_cut(int batch, int queries, int H, int Hkv, int d, int dtype, int max_kv) {
  const int rows = queries * (H / Hkv), need = (rows + 15) / 16;
  TreeCut cut;
  cut.shared = need > 2;
  cut.tiles = cut.shared ? (need <= 8 ? 8 : 16) : need;
  cut.groups = (need + cut.tiles - 1) / cut.tiles;
  const int ck = dtype == SPECDEC_BF16 ? 32 : 16, chunks = (max_kv + ck - 1) / ck;
  const int64_t units = (int64_t)batch * Hkv * cut.groups;
  // two workgroups a compute unit, what the registers of most variants let in at
  // once, and four chunks a wave, below which the second launch costs more than it
  // gives (measured: 8 rows of 32 nodes at 4096 keys 55.9 / 56.8 / 64.5 us in 1 / 2 /
  // 4 splits, one row of 16 at 300 keys 7.6 / 9.8 in 1 / 2, four fp32 rows of 13 at
  // 1500 keys 34.5 / 26.4 / 26.6 / 34.8 in 1 / 2 / 4 / 8)
  int64_t splits = (cut.tiles == 16 ? 256 : 512) / units;
  const int least = cut.shared ? 8 : 4 * kTreeWaves;
  splits = splits < chunks / least ? splits : chunks / least;
  cut.splits = (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
  return cut;
}
inline int64_t tree_floats(const TreeCut &cut, int batch, int Hkv, int d) {
  return cut.splits > 1 ? (int64_t)batch * Hkv * cut.splits * cut.rows() * (d + 2) : 0;
}

// ------------------------------------------------------------------ commit --
struct CommitArgs {
  const int64_t *tokens, *sampled;
  int64_t tokens_stride, sampled_stride;
  const int32_t *parents;
  int64_t parents_stride;
  const int32_t *meta;
  int batch, nodes, room;
  int64_t *verdict;  // [nodes + 1, batch]
  int32_t *path;     // [batch, nodes]
  // the append; layers = 0 for the walk alone
  const void *qkv;
  int layers;
  int64_t layer_stride, batch_stride, token_stride;
  const float *cos_t, *sin_t;
  int positions, H, Hkv, d, bs;
  void *k_pool, *v_pool;  // [layers, num_blocks, Hkv, bs, d], [layers, num_blocks, Hkv, d, bs]
  int num_blocks;
  const int32_t *tables;
  int64_t table_stride;
  int table_rows, table_cols;
};

constexpr int kCommitThreads = 256;
constexpr int kCommitHeads = 8;  // kv heads of a workgroup

// Grid (batch, layers or 1, groups of kv heads).  Every workgroup walks its row's
// tree, a step a path node, by ballots of one wave; the first of layer 0 writes
// the verdict; each appends the path's keys and values of its heads to its layer.
// VEC: a thread takes 16 bytes of each half of a head's k and v.  The path's nodes
// are its threads' fastest index, so that neighbours write neighbouring slots of a
// V row, whose elements lie a block apart from dim to dim: those 2-byte stores are
// what it is bound by: some 28 MB of 32 rows, 24 layers of 32 heads of 64, leave as 79
// MB, 41 us (one element of one head a thread at a time took 86).
template <typename T, bool VEC> __global__ __launch_bounds__(kCommitThreads) void tree_commit_kernel(CommitArgs a) {
  const int b = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x, lane = tid & (kWave - 1);
  __shared__ int64_t tokens[kTreeMaxNodes], sampled[kTreeMaxNodes];
  __shared__ int32_t parents[kTreeMaxNodes], way[kTreeMaxNodes], block_of[kTreeMaxNodes];
  __shared__ int n_way;
  const int row = a.meta[b], past = a.meta[a.batch + b], live = min(a.meta[2 * a.batch + b], a.nodes);
  if (tid < live) {
    tokens[tid] = a.tokens[b * a.tokens_stride + tid];
    sampled[tid] = a.sampled[b * a.sampled_stride + tid];
    parents[tid] = a.parents[b * a.parents_stride + tid];
  }
  // the blocks of the slots that the path may take; it ends before the first that is none
  int room = min(a.room, live);
  if (tid == 0) n_way = room;
  __syncthreads();
  if (a.layers > 0 && tid < room) {
    const int64_t pos = (int64_t)past + tid;
    const bool in = row >= 0 && row < a.table_rows && past >= 0 && pos < (int64_t)a.table_cols * a.bs && pos < a.positions;
    const int id = in ? a.tables[row * a.table_stride + pos / a.bs] : -1;
    block_of[tid] = id;
    if (id < 0 || id >= a.num_blocks) atomicMin(&n_way, tid);
  }
  __syncthreads();
  room = n_way;
  __syncthreads();
  if (tid < kWave) {
    int n = 0, cur = 0;
    if (room > 0) {
      if (lane == 0) way[0] = 0;
      n = 1;
      while (n < room) {
        const int64_t want = sampled[cur];
        int next = -1;
        for (int c0 = (cur + 1) & ~(kWave - 1); c0 < live && next < 0; c0 += kWave) {
          const int c = c0 + lane;
          const uint64_t hit = __ballot(c > cur && c < live && parents[c] == cur && tokens[c] == want);
          if (hit) next = c0 + __ffsll((unsigned long long)hit) - 1;
        }
        if (next < 0) break;
        if (lane == 0) way[n] = next;
        cur = next;
        ++n;
      }
    }
    if (lane == 0) n_way = n;
  }
  __syncthreads();
  const int n = n_way;
  if (layer == 0 && blockIdx.z == 0) {
    for (int j = tid; j < a.nodes; j += kCommitThreads) {
      a.path[(int64_t)b * a.nodes + j] = j < n ? way[j] : -1;
      if (j > 0) a.verdict[(int64_t)(j + 1) * a.batch + b] = j < n ? tokens[way[j]] : -1;
    }
    if (tid == 0) {
      a.verdict[b] = n - 1;
      a.verdict[a.batch + b] = n > 0 ? sampled[way[n - 1]] : -1;
    }
  }
  if (a.layers == 0) return;
  const T *rows = (const T *)a.qkv + layer * a.layer_stride + b * a.batch_stride;
  const int half = a.d / 2, h0 = blockIdx.z * kCommitHeads, heads = min(kCommitHeads, a.Hkv - h0);
  const int64_t tile = (int64_t)a.bs * a.d, pool = (int64_t)layer * a.num_blocks * a.Hkv * tile;
  T *kp = (T *)a.k_pool + pool, *vp = (T *)a.v_pool + pool;
  constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;
  const int pieces = half / E;
  for (int i = tid; i < heads * pieces * n; i += kCommitThreads) {
    const int j = i % n, h = h0 + i / n / pieces, x = i / n % pieces * E;
    const int pos = past + j, slot = pos % a.bs;
    const T *k = rows + way[j] * a.token_stride + (int64_t)(a.H + h) * a.d + x, *v = k + (int64_t)a.Hkv * a.d;
    const float *cp = a.cos_t + (int64_t)pos * half + x, *sp = a.sin_t + (int64_t)pos * half + x;
    const int64_t at = ((int64_t)block_of[j] * a.Hkv + h) * tile;
    T *ko = kp + at + (int64_t)slot * a.d + x, *vo = vp + at + (int64_t)x * a.bs + slot;
    if constexpr (VEC) {
      u32x4 lo = *(const u32x4 *)k, hi = *(const u32x4 *)(k + half);
      const u32x4 v1 = *(const u32x4 *)v, v2 = *(const u32x4 *)(v + half);
      float c[E], s[E];
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        *(f32x4 *)&c[e] = *(const f32x4 *)(cp + e);
        *(f32x4 *)&s[e] = *(const f32x4 *)(sp + e);
      }
      tree_rotate<E>(lo, hi, c, s, true);
      *(u32x4 *)ko = lo;
      *(u32x4 *)(ko + half) = hi;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (sizeof(T) == 2) {
          ((uint16_t *)vo)[(int64_t)e * a.bs] = (uint16_t)(v1[e / 2] >> 16 * (e % 2));
          ((uint16_t *)vo)[(int64_t)(half + e) * a.bs] = (uint16_t)(v2[e / 2] >> 16 * (e % 2));
        } else {
          ((uint32_t *)vo)[(int64_t)e * a.bs] = v1[e];
          ((uint32_t *)vo)[(int64_t)(half + e) * a.bs] = v2[e];
        }
      }
    } else {
      float y1, y2;
      rope_pair(to_f32(k[0]), to_f32(k[half]), cp[0], sp[0], y1, y2);
      ko[0] = from_f32<T>(y1);
      ko[half] = from_f32<T>(y2);
      vo[0] = v[0];
      vo[(int64_t)half * a.bs] = v[half];
    }
  }
}

template <typename T> int launch_tree_commit(const CommitArgs &a, hipStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  const auto aligned = [](const void *p) { return (uintptr_t)p % 16 == 0; };
  const dim3 grid((unsigned)a.batch, (unsigned)(a.layers > 0 ? a.layers : 1),
                  (unsigned)(a.layers > 0 ? (a.Hkv + kCommitHeads - 1) / kCommitHeads : 1));
  if (a.d / 2 % E == 0 && aligned(a.qkv) && a.layer_stride % E == 0 && a.batch_stride % E == 0 && a.token_stride % E == 0 &&
      aligned(a.cos_t) && aligned(a.sin_t) && aligned(a.k_pool) && aligned(a.v_pool))
    tree_commit_kernel<T, true><<<grid, kCommitThreads, 0, s>>>(a);
  else
    tree_commit_kernel<T, false><<<grid, kCommitThreads, 0, s>>>(a);
  return launch_status();
}

template <typename T, int D> int launch_tree_tiles(const TreeArgs &a, const TreeCut &cut, float *ws, hipStream_t s) {
  const int64_t units = (int64_t)a.batch * a.Hkv * cut.splits;
  const int64_t grid = cut.groups > 1 ? (units + 7) / 8 * 8 * cut.groups : units;
  if (grid > INT32_MAX) return SPECDEC_EUNSUPPORTED;
  int shift = 0;
  while (1 << shift < a.bs) ++shift;
  if (1 << shift != a.bs) shift = -1;
  const dim3 block(kTreeWaves * kWave);
  constexpr int NT = D / 64;  // of 8 tiles: what the registers of four waves a SIMD hold, or of two
  if (cut.tiles == 16) tree_attention_shared_kernel<T, D, 8, 2><<<(unsigned)grid, 8 * kWave, 0, s>>>(a, cut, shift, ws);
  else if (cut.tiles == 8)
    tree_attention_shared_kernel<T, D, 8 / NT, NT><<<(unsigned)grid, 8 / NT * kWave, 0, s>>>(a, cut, shift, ws);
  else if (cut.tiles == 1) tree_attention_kernel<T, D, 1><<<(unsigned)grid, block, 0, s>>>(a, cut, shift, ws);
  else tree_attention_kernel<T, D, 2><<<(unsigned)grid, block, 0, s>>>(a, cut, shift, ws);
  if (cut.splits > 1) {
    const int rows = (a.nodes - a.first) * (a.H / a.Hkv), per = 256 / (D / 4);
    tree_fold_kernel<T, D><<<dim3((rows + per - 1) / per, a.Hkv, a.batch), 256, 0, s>>>(a, cut, ws);
  }
  return launch_status();
}

template <typename T, int D>
int launch_tree_attention(const TreeArgs &a, int dtype, int max_kv, float *ws, int64_t floats, hipStream_t s) {
  // pieces of 16 bytes: rows, tables and pools aligned, blocks of whole pieces
  constexpr int EPL = 16 / (int)sizeof(T);
  const auto aligned = [](const void *p) { return (uintptr_t)p % 16 == 0; };
  if (aligned(a.qkv) && a.batch_stride % EPL == 0 && a.token_stride % EPL == 0 && aligned(a.cos_t) && aligned(a.sin_t) &&
      aligned(a.k_pool) && aligned(a.v_pool) && a.bs % EPL == 0) {
    TreeCut cut = tree_cut(a.batch, a.nodes - a.first, a.H, a.Hkv, D, dtype, max_kv);
    if (tree_floats(cut, a.batch, a.Hkv, D) > floats || !ws || !aligned(ws)) cut.splits = 1;
    return launch_tree_tiles<T, D>(a, cut, ws, s);
  }
  const dim3 grid((unsigned)(a.nodes - a.first), (unsigned)a.H, (unsigned)a.batch);
  tree_attention_any_kernel<T, D><<<grid, kWave, 0, s>>>(a);
  return launch_status();
}

}  // namespace specdec

using namespace specdec;

SPECDEC_API int specdec_tree_attention_workspace(int32_t batch, int32_t nodes, int32_t first, int32_t n_heads,
                                                 int32_t n_kv_heads, int32_t head_dim, int dtype, int32_t block_size,
                                                 int32_t max_kv_len, int64_t *floats) {
  if (batch < 0 || nodes < 0 || first < 0 || first > nodes || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads ||
      head_dim <= 0 || block_size <= 0 || max_kv_len < 0 || !floats)
    return SPECDEC_EINVAL;
  if (head_dim != 64 && head_dim != 128) return SPECDEC_EUNSUPPORTED;
  if (dtype != SPECDEC_F32 && dtype != SPECDEC_BF16) return SPECDEC_EUNSUPPORTED;
  if (nodes > kTreeMaxNodes) return SPECDEC_EUNSUPPORTED;
  *floats = batch == 0 || nodes == first ? 0
            : tree_floats(tree_cut(batch, nodes - first, n_heads, n_kv_heads, head_dim, dtype, max_kv_len), batch,
                          n_kv_heads, head_dim);
  return SPECDEC_OK;
}

SPECDEC_API int specdec_tree_attention(const void *qkv, int dtype, int64_t batch_stride, int64_t token_stride,
                                       const float *cos_table, const float *sin_table, int64_t max_positions,
                                       const void *k_pool, const void *v_pool, int64_t num_blocks, const int32_t *tables,
                                       int64_t table_stride, int32_t table_rows, int32_t table_cols,
                                       const int32_t *meta, const int64_t *mask, int64_t mask_batch_stride,
                                       int64_t mask_row_stride, const int32_t *depth, int64_t depth_batch_stride,
                                       int32_t batch, int32_t nodes, int32_t first, int32_t n_heads,
                                       int32_t n_kv_heads, int32_t head_dim, int32_t block_size, float scale,
                                       int32_t max_kv_len, float *workspace, int64_t workspace_floats, void *out,
                                       int64_t out_batch_stride, int64_t out_token_stride, void *stream) {
  if (batch < 0 || nodes < 0 || first < 0 || first > nodes || n_heads <= 0 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads || block_size <= 0 || max_positions <= 0 || num_blocks < 0 || table_rows < 0 ||
      table_cols < 0 || table_stride < table_cols || max_kv_len < 0 || workspace_floats < 0)
    return SPECDEC_EINVAL;
  if (head_dim != 64 && head_dim != 128) return SPECDEC_EUNSUPPORTED;
  if (dtype != SPECDEC_F32 && dtype != SPECDEC_BF16) return SPECDEC_EUNSUPPORTED;
  if (nodes > kTreeMaxNodes || batch > 65535 || n_heads > 65535 || num_blocks > INT32_MAX || max_positions > INT32_MAX)
    return SPECDEC_EUNSUPPORTED;
  if (batch == 0 || nodes == first) return SPECDEC_OK;
  const int64_t row = (int64_t)(n_heads + 2 * n_kv_heads) * head_dim, orow = (int64_t)n_heads * head_dim;
  if ((nodes > 1 && token_stride < row) || (nodes - first > 1 && out_token_stride < orow)) return SPECDEC_EINVAL;
  if (!qkv || !cos_table || !sin_table || !meta || !mask || !depth || !out) return SPECDEC_EINVAL;
  // a cache of no block or no table can hold rows of no cached position alone
  if (num_blocks == 0 || table_rows == 0) table_cols = 0;
  if (table_cols > 0 && (!k_pool || !v_pool || !tables)) return SPECDEC_EINVAL;
  TreeArgs a{qkv, batch_stride, token_stride, cos_table, sin_table, (int)max_positions, k_pool, v_pool, (int)num_blocks,
             tables, table_stride, table_rows, table_cols, meta, mask, mask_batch_stride, mask_row_stride, depth,
             depth_batch_stride, batch, nodes, first, n_heads, n_kv_heads, block_size, scale, out, out_batch_stride,
             out_token_stride};
  const hipStream_t s = as_stream(stream);
  if (dtype == SPECDEC_F32)
    return head_dim == 64 ? launch_tree_attention<float, 64>(a, dtype, max_kv_len, workspace, workspace_floats, s)
                          : launch_tree_attention<float, 128>(a, dtype, max_kv_len, workspace, workspace_floats, s);
  return head_dim == 64
             ? launch_tree_attention<__hip_bfloat16, 64>(a, dtype, max_kv_len, workspace, workspace_floats, s)
             : launch_tree_attention<__hip_bfloat16, 128>(a, dtype, max_kv_len, workspace, workspace_floats, s);
}

SPECDEC_API int specdec_tree_commit(const int64_t *tokens, int64_t tokens_stride, const int32_t *parents,
                                    int64_t parents_stride, const int64_t *sampled, int64_t sampled_stride,
                                    const int32_t *meta, int32_t batch, int32_t nodes, int32_t room, int64_t *verdict,
                                    int32_t *path, const void *qkv, int dtype, int32_t layers, int64_t layer_stride,
                                    int64_t batch_stride, int64_t token_stride, const float *cos_table,
                                    const float *sin_table, int64_t max_positions, int32_t n_heads, int32_t n_kv_heads,
                                    int32_t head_dim, int32_t block_size, void *k_pool, void *v_pool,
                                    int64_t num_blocks, const int32_t *tables, int64_t table_stride, int32_t table_rows,
                                    int32_t table_cols, void *stream) {
  if (batch < 0 || nodes <= 0 || room <= 0 || layers < 0) return SPECDEC_EINVAL;
  if (nodes > kTreeMaxNodes || layers > 65535) return SPECDEC_EUNSUPPORTED;
  if (batch == 0) return SPECDEC_OK;
  if (!tokens || !parents || !sampled || !meta || !verdict || !path) return SPECDEC_EINVAL;
  CommitArgs a{tokens, sampled, tokens_stride, sampled_stride, parents, parents_stride, meta, batch, nodes, room, verdict,
               path, qkv, layers, layer_stride, batch_stride, token_stride, cos_table, sin_table, (int)max_positions,
               n_heads, n_kv_heads, head_dim, block_size, k_pool, v_pool, (int)num_blocks, tables, table_stride,
               table_rows, table_cols};
  if (layers > 0) {
    if (n_heads < 0 || n_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || max_positions <= 0 || num_blocks <= 0 ||
        table_rows <= 0 || table_cols <= 0 || table_stride < table_cols)
      return SPECDEC_EINVAL;
    if (nodes > 1 && token_stride < (int64_t)(n_heads + 2 * n_kv_heads) * head_dim) return SPECDEC_EINVAL;
    if (!qkv || !cos_table || !sin_table || !k_pool || !v_pool || !tables) return SPECDEC_EINVAL;
    if (head_dim % 2 || head_dim > 512 || n_kv_heads > 4096 || num_blocks > INT32_MAX || max_positions > INT32_MAX)
      return SPECDEC_EUNSUPPORTED;
    if (dtype != SPECDEC_F32 && dtype != SPECDEC_BF16) return SPECDEC_EUNSUPPORTED;
  }
  return layers > 0 && dtype == SPECDEC_F32 ? launch_tree_commit<float>(a, as_stream(stream))
                                            : launch_tree_commit<__hip_bfloat16>(a, as_stream(stream));
}
