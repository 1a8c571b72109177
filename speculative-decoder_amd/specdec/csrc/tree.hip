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
// any block size, stride and alignment; what it is bound by is its scattered
// reads.
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

// Grid (batch, layers or 1).  Every workgroup walks its row's tree, a step a
// path node, by ballots of one wave; that of layer 0 writes the verdict; each
// appends the path's keys and values to its layer.
template <typename T> __global__ __launch_bounds__(kCommitThreads) void tree_commit_kernel(CommitArgs a) {
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
  if (layer == 0) {
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
  const int half = a.d / 2, per_token = a.Hkv * half;
  const int64_t tile = (int64_t)a.bs * a.d, pool = (int64_t)layer * a.num_blocks * a.Hkv * tile;
  T *kp = (T *)a.k_pool + pool, *vp = (T *)a.v_pool + pool;
  for (int e = tid; e < n * per_token; e += kCommitThreads) {
    const int j = e / per_token, h = e % per_token / half, x = e % half;
    const int pos = past + j, slot = pos % a.bs;
    const T *k = rows + way[j] * a.token_stride + (int64_t)(a.H + h) * a.d, *v = k + (int64_t)a.Hkv * a.d;
    const float c = a.cos_t[(int64_t)pos * half + x], s = a.sin_t[(int64_t)pos * half + x];
    float y1, y2;
    rope_pair(to_f32(k[x]), to_f32(k[x + half]), c, s, y1, y2);
    const int64_t at = ((int64_t)block_of[j] * a.Hkv + h) * tile;
    kp[at + (int64_t)slot * a.d + x] = from_f32<T>(y1);
    kp[at + (int64_t)slot * a.d + x + half] = from_f32<T>(y2);
    vp[at + (int64_t)x * a.bs + slot] = v[x];
    vp[at + (int64_t)(x + half) * a.bs + slot] = v[x + half];
  }
}

template <typename T> int launch_tree_attention(const TreeArgs &a, int d, hipStream_t s) {
  const dim3 grid((unsigned)(a.nodes - a.first), (unsigned)a.H, (unsigned)a.batch);
  if (d == 64) tree_attention_any_kernel<T, 64><<<grid, kWave, 0, s>>>(a);
  else tree_attention_any_kernel<T, 128><<<grid, kWave, 0, s>>>(a);
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
  (void)dtype;
  *floats = 0;
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
  (void)workspace;
  TreeArgs a{qkv, batch_stride, token_stride, cos_table, sin_table, (int)max_positions, k_pool, v_pool, (int)num_blocks,
             tables, table_stride, table_rows, table_cols, meta, mask, mask_batch_stride, mask_row_stride, depth,
             depth_batch_stride, batch, nodes, first, n_heads, n_kv_heads, block_size, scale, out, out_batch_stride,
             out_token_stride};
  if (dtype == SPECDEC_F32) return launch_tree_attention<float>(a, head_dim, as_stream(stream));
  return launch_tree_attention<__hip_bfloat16>(a, head_dim, as_stream(stream));
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
  const dim3 grid((unsigned)batch, (unsigned)(layers > 0 ? layers : 1)), block(kCommitThreads);
  if (layers > 0 && dtype == SPECDEC_F32) tree_commit_kernel<float><<<grid, block, 0, as_stream(stream)>>>(a);
  else tree_commit_kernel<__hip_bfloat16><<<grid, block, 0, as_stream(stream)>>>(a);
  return launch_status();
}
