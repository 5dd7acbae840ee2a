// (7) Attention of a tree of drafted tokens over cache rows and the tree itself.
//
// A verification step asks for the attention of T drafted tokens of a request
// at once. They share the request's selected cache rows, so the T * G query
// rows of a KV head (G query heads in its group) form one matrix: S = Q K^T /
// sqrt(D), a softmax along the keys, O = P V. The keys of a request are one
// list: its valid cache rows, then its nodes; key i < valid is the pool row
// rows[i], key valid + j is node j. Every query row sees every cache row;
// mask[t] says which nodes node t sees.
//
// A block serves (request, KV head, a tile of query rows, a split of the key
// list) with the running maximum m, the sum l of exp(s - m) and the
// unnormalised O in fp32. With one split it writes the result; with more it
// leaves (O, m, l) in the workspace and a second launch joins the splits:
// O = sum_i exp(m_i - m) O_i / sum_i exp(m_i - m) l_i.
#include <math.h>

#include "common.cuh"
#include "hisparse_verify.h"

namespace hs {
namespace {

constexpr int kTreeMaxNodes = 64;
constexpr int kTreeMaxDim = 256;
constexpr int kTreeMaxSplits = 64;

struct TreeParams {
  int batch, nodes;
  const void *query, *key, *value;
  int64_t q_batch_stride, q_node_stride, kv_batch_stride, kv_node_stride;
  const int64_t *mask;
  const int32_t *node_counts;
  const void *pool;
  int64_t pool_blocks;
  const int64_t *rows;
  int64_t rows_batch_stride, count;
  const int32_t *counts;
  void *out;
  int q_heads, kv_heads, head_dim, page_size, page_shift;  // page_shift: log2 or -1
  int groups;           // query heads of a KV head
  int splits;
  float scale_log2;     // log2(e) / sqrt(head_dim): scores are kept in powers of two
  float *partials;      // [batch][kv_heads][nodes * groups][splits][head_dim + 2]
  int32_t *status;
};

__device__ __forceinline__ int64_t rows_of(const TreeParams &p, int b) {
  if (p.counts == nullptr) return p.count;
  const int64_t n = p.counts[b];
  return n < 0 ? 0 : (n > p.count ? p.count : n);
}
__device__ __forceinline__ int nodes_of(const TreeParams &p, int b) {
  if (p.node_counts == nullptr) return p.nodes;
  const int n = p.node_counts[b];
  return n < 0 ? 0 : (n > p.nodes ? p.nodes : n);
}

// Element offset in the pool of physical row `row` of the K plane (the V plane
// is page_size rows further); -1 for a row that is padding or outside the pool.
__device__ __forceinline__ int64_t row_offset(const TreeParams &p, int64_t row, int64_t row_elems) {
  if (row < 0) return -1;
  int64_t block, within;
  if (p.page_shift >= 0) {
    block = row >> p.page_shift;
    within = row & (p.page_size - 1);
  } else {
    block = row / p.page_size;
    within = row - block * p.page_size;
  }
  if (block >= p.pool_blocks) {
    flag(p.status, HS_DEV_ROW_OUT_OF_RANGE);
    return -1;
  }
  return (block * 2 * p.page_size + within) * row_elems;
}

__device__ __forceinline__ float *partial_of(const TreeParams &p, int b, int kh, int r, int split) {
  return p.partials + ((((int64_t)b * p.kv_heads + kh) * (p.nodes * p.groups) + r) * p.splits +
                       split) * (p.head_dim + 2);
}

// ---- fp32 arithmetic: every type, head_dim and alignment -------------------------------
// 128 threads over a tile of 32 query rows and 64 keys, operands widened to fp32
// in shared memory. For the scores a thread holds 4 rows x 4 keys, for the output
// 4 rows x 4 NJ elements, so that four products follow each shared-memory word.
constexpr int kSimtThreads = 128;
constexpr int kSimtRows = 32;
constexpr int kSimtKeys = 64;
constexpr int kSimtPPitch = kSimtKeys + 4;

template <int NJ> struct SimtShape {
  static constexpr int dim = 64 * NJ;     // head_dim rounded up, the rest zero
  static constexpr int pitch = dim + 4;   // floats between rows
  static constexpr size_t bytes =
      sizeof(float) * ((kSimtRows + 2 * kSimtKeys) * pitch + kSimtRows * kSimtPPitch);
};

template <typename T, int NJ>
__global__ void __launch_bounds__(kSimtThreads) tree_simt_kernel(TreeParams p) {
  using Shape = SimtShape<NJ>;
  constexpr int dim = Shape::dim, pitch = Shape::pitch;
  extern __shared__ __align__(16) float smem[];
  float *sq = smem, *sk = sq + kSimtRows * pitch, *sv = sk + kSimtKeys * pitch;
  float *sp = sv + kSimtKeys * pitch;
  __shared__ int64_t s_src[kSimtKeys];  // element offset of a key's K; see below
  __shared__ uint64_t s_mask[kSimtRows];
  const int tid = threadIdx.x, split = blockIdx.x;
  const int tiles = (int)ceil_div(p.nodes * p.groups, kSimtRows);
  const int kh = blockIdx.y / tiles, r0 = blockIdx.y % tiles * kSimtRows, b = blockIdx.z;
  const int D = p.head_dim, G = p.groups;
  const int n_nodes = nodes_of(p, b), live = n_nodes * G;  // query rows with a result
  const int64_t valid = rows_of(p, b), total = valid + n_nodes;
  const int64_t chunk = ceil_div(ceil_div(total, p.splits), kSimtKeys) * kSimtKeys;
  const int64_t begin = split * chunk, end = min(total, begin + chunk);
  const int tx = tid & 15, ty = tid >> 4;  // keys / elements; rows 4 ty .. 4 ty + 3

  const T *query = static_cast<const T *>(p.query) + b * p.q_batch_stride;
  for (int i = tid; i < kSimtRows * dim; i += kSimtThreads) {
    const int r = i / dim, d = i % dim, row = r0 + r;
    sq[r * pitch + d] =
        row < live && d < D
            ? to_f32(query[row / G * p.q_node_stride + (kh * G + row % G) * (int64_t)D + d])
            : 0.f;
  }
  if (tid < kSimtRows) {
    const int row = r0 + tid;
    uint64_t m = row < live ? (uint64_t)p.mask[(int64_t)b * p.nodes + row / G] : 0;
    s_mask[tid] = n_nodes < 64 ? m & ((1ull << n_nodes) - 1) : m;
  }
  float m[4], l[4], acc[4][4 * NJ];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < 4 * NJ; ++j) acc[i][j] = 0.f;
  }
  const int64_t row_elems = (int64_t)p.kv_heads * D;
  const T *pool = static_cast<const T *>(p.pool) + (int64_t)kh * D;
  const T *key = static_cast<const T *>(p.key) + b * p.kv_batch_stride + (int64_t)kh * D;
  const T *value = static_cast<const T *>(p.value) + b * p.kv_batch_stride + (int64_t)kh * D;
  const int64_t *rows = p.rows + b * p.rows_batch_stride;

  for (int64_t k0 = begin; k0 < end; k0 += kSimtKeys) {
    __syncthreads();
    // where each key lives: >= 0 in the pool, -1 nowhere, -2 - j node j
    if (tid < kSimtKeys) {
      const int64_t i = k0 + tid;
      s_src[tid] = i >= end ? -1
                   : i < valid ? row_offset(p, rows[i], row_elems)
                               : -2 - (i - valid);
    }
    __syncthreads();
    for (int i = tid; i < kSimtKeys * dim; i += kSimtThreads) {
      const int k = i / dim, d = i % dim;
      const int64_t src = s_src[k];
      float kx = 0.f, vx = 0.f;
      if (d < D && src >= 0) {
        kx = to_f32(pool[src + d]);
        vx = to_f32(pool[src + p.page_size * row_elems + d]);
      } else if (d < D && src < -1) {
        kx = to_f32(key[(-2 - src) * p.kv_node_stride + d]);
        vx = to_f32(value[(-2 - src) * p.kv_node_stride + d]);
      }
      sk[k * pitch + d] = kx;
      sv[k * pitch + d] = vx;
    }
    __syncthreads();
    float s[4][4];  // rows 4 ty + i, keys tx + 16 j
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    for (int d = 0; d < dim; d += 4) {
      float4 q4[4], k4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q4[i] = *reinterpret_cast<const float4 *>(&sq[(4 * ty + i) * pitch + d]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        k4[j] = *reinterpret_cast<const float4 *>(&sk[(tx + 16 * j) * pitch + d]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = fmaf(q4[i].x, k4[j].x, fmaf(q4[i].y, k4[j].y,
                    fmaf(q4[i].z, k4[j].z, fmaf(q4[i].w, k4[j].w, s[i][j]))));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t src = s_src[tx + 16 * j];
        const bool seen = src >= 0 || (src < -1 && (s_mask[4 * ty + i] >> (-2 - src) & 1));
        s[i][j] = seen ? s[i][j] * p.scale_log2 : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
      const float m_new = fmaxf(m[i], top);
      const float alpha = m[i] == -INFINITY ? 0.f : exp2f(m[i] - m_new);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = s[i][j] == -INFINITY ? 0.f : exp2f(s[i][j] - m_new);
        sum += w;
        sp[(4 * ty + i) * kSimtPPitch + tx + 16 * j] = w;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
      l[i] = l[i] * alpha + sum;
      m[i] = m_new;
#pragma unroll
      for (int j = 0; j < 4 * NJ; ++j) acc[i][j] *= alpha;
    }
    __syncwarp();  // a row's probabilities are written and read by the same half warp
    for (int k = 0; k < kSimtKeys; ++k) {
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = sp[(4 * ty + i) * kSimtPPitch + k];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const float4 v4 = *reinterpret_cast<const float4 *>(&sv[k * pitch + 4 * tx + 64 * j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // a pair that is not seen takes no part even where its value is NaN or infinite
          if (w[i] != 0.f) {
            acc[i][4 * j] = fmaf(w[i], v4.x, acc[i][4 * j]);
            acc[i][4 * j + 1] = fmaf(w[i], v4.y, acc[i][4 * j + 1]);
            acc[i][4 * j + 2] = fmaf(w[i], v4.z, acc[i][4 * j + 2]);
            acc[i][4 * j + 3] = fmaf(w[i], v4.w, acc[i][4 * j + 3]);
          }
        }
      }
    }
  }
  // rows of padded nodes: one split writes their zeros
  const int rows_all = p.nodes * G;
  T *out = static_cast<T *>(p.out) + (int64_t)b * p.nodes * p.q_heads * D;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + 4 * ty + i;
    if (row >= rows_all) continue;
    if (p.splits == 1) {
      const float inv = l[i] > 0.f || l[i] != l[i] ? 1.f / l[i] : 0.f;
      T *o = out + (int64_t)(row / G) * p.q_heads * D + (int64_t)(kh * G + row % G) * D;
#pragma unroll
      for (int j = 0; j < 4 * NJ; ++j) {
        const int d = 4 * tx + 64 * (j / 4) + j % 4;
        if (d < D) o[d] = from_f32<T>(row < live ? acc[i][j] * inv : 0.f);
      }
    } else {
      float *o = partial_of(p, b, kh, row, split);
#pragma unroll
      for (int j = 0; j < 4 * NJ; ++j) {
        const int d = 4 * tx + 64 * (j / 4) + j % 4;
        if (d < D) o[d] = acc[i][j];
      }
      if (tx == 0) {
        o[D] = m[i];
        o[D + 1] = l[i];
      }
    }
  }
}

// ---- joining the splits ------------------------------------------------------------------
// One block for each (node, query head, request); thread d sums element d.
template <typename T>
__global__ void __launch_bounds__(kTreeMaxDim) tree_merge_kernel(TreeParams p) {
  const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z, d = threadIdx.x;
  const int kh = h / p.groups, row = t * p.groups + h % p.groups, D = p.head_dim;
  if (d >= D) return;
  float m = -INFINITY, l = 0.f, o = 0.f;
  if (t < nodes_of(p, b)) {
    const float *first = partial_of(p, b, kh, row, 0);
    for (int s = 0; s < p.splits; ++s) {
      const float *part = first + (int64_t)s * (D + 2);
      const float ms = part[D], ls = part[D + 1];
      if (ls == 0.f) continue;  // a split that saw nothing left no sums
      const float m_new = fmaxf(m, ms);
      const float f = m == -INFINITY ? 0.f : exp2f(m - m_new), g = exp2f(ms - m_new);
      l = l * f + ls * g;
      o = o * f + part[d] * g;
      m = m_new;
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  static_cast<T *>(p.out)[(((int64_t)b * p.nodes + t) * p.q_heads + h) * D + d] =
      from_f32<T>(o * inv);
}

// Splits of the key list: enough blocks for two on every SM, no split shorter
// than two tiles of keys.
int tree_splits(int batch, int nodes, int q_heads, int kv_heads, int64_t count) {
  const int64_t tiles = ceil_div((int64_t)nodes * (q_heads / kv_heads), kSimtRows);
  int64_t s = ceil_div((int64_t)2 * sm_count(), (int64_t)batch * kv_heads * tiles);
  const int64_t longest = ceil_div(count + nodes, 2 * kSimtKeys);
  if (s > longest) s = longest;
  if (s > kTreeMaxSplits) s = kTreeMaxSplits;
  return s < 1 ? 1 : (int)s;
}

template <typename T, int NJ> int launch_simt(const TreeParams &p, cudaStream_t s) {
  auto kernel = tree_simt_kernel<T, NJ>;
  const size_t bytes = SimtShape<NJ>::bytes;
  if (int e = reserve_smem(reinterpret_cast<const void *>(kernel), bytes, "attend_tree")) return e;
  const int64_t tiles = ceil_div((int64_t)p.nodes * p.groups, kSimtRows);
  const dim3 grid((unsigned)p.splits, (unsigned)(p.kv_heads * tiles), (unsigned)p.batch);
  kernel<<<grid, kSimtThreads, bytes, s>>>(p);
  if (int e = check_launch("tree_simt_kernel")) return e;
  if (p.splits == 1) return HS_OK;
  const dim3 merge((unsigned)p.nodes, (unsigned)p.q_heads, (unsigned)p.batch);
  tree_merge_kernel<T><<<merge, (unsigned)(ceil_div(p.head_dim, 32) * 32), 0, s>>>(p);
  return check_launch("tree_merge_kernel");
}

template <typename T> int launch(const TreeParams &p, cudaStream_t s) {
  switch (ceil_div(p.head_dim, 64)) {
    case 1: return launch_simt<T, 1>(p, s);
    case 2: return launch_simt<T, 2>(p, s);
    case 3: return launch_simt<T, 3>(p, s);
    default: return launch_simt<T, 4>(p, s);
  }
}

}  // namespace
}  // namespace hs

extern "C" size_t hs_attend_tree_workspace_bytes(int batch, int nodes, int q_heads, int kv_heads,
                                                 int head_dim, int64_t count, int dtype) {
  using namespace hs;
  (void)dtype;
  if (batch < 1 || nodes < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || count < 0)
    return 0;
  const int splits = tree_splits(batch, nodes, q_heads, kv_heads, count);
  if (splits == 1) return 0;
  return (size_t)batch * nodes * q_heads * splits * (head_dim + 2) * sizeof(float);
}

extern "C" int hs_attend_tree(int batch, int nodes, const void *query, int64_t query_batch_stride,
                              int64_t query_node_stride, const void *key, const void *value,
                              int64_t kv_batch_stride, int64_t kv_node_stride, int dtype,
                              const int64_t *mask, const int32_t *node_counts, const void *pool,
                              int64_t pool_blocks, const int64_t *rows, int64_t rows_batch_stride,
                              int64_t count, const int32_t *counts, void *out, int q_heads,
                              int kv_heads, int head_dim, int page_size, void *workspace,
                              size_t workspace_bytes, int32_t *device_status, hs_stream stream) {
  using namespace hs;
  if (batch < 0 || nodes < 0 || kv_heads < 1 || q_heads < 1 || head_dim < 1 || page_size < 1 ||
      pool_blocks < 0 || count < 0)
    return set_error(HS_ERR_INVALID_ARGUMENT, "attend_tree: invalid sizes");
  if (q_heads % kv_heads)
    return set_error(HS_ERR_INVALID_ARGUMENT, "query GQA/device mismatch");
  if (nodes > kTreeMaxNodes)
    return set_error(HS_ERR_UNSUPPORTED, "attend_tree: %d nodes > %d are not supported", nodes,
                     kTreeMaxNodes);
  if (head_dim > kTreeMaxDim)
    return set_error(HS_ERR_UNSUPPORTED, "attend_tree: head_dim %d > %d is not supported",
                     head_dim, kTreeMaxDim);
  if (dtype != HS_FLOAT32 && dtype != HS_FLOAT16 && dtype != HS_BFLOAT16)
    return set_error(HS_ERR_INVALID_ARGUMENT, "attend_tree: invalid dtype %d", dtype);
  if (batch == 0 || nodes == 0) return HS_OK;
  if (batch > 65535 || q_heads > 32767 || count > 0x7fffff00)
    return set_error(HS_ERR_UNSUPPORTED, "attend_tree: batch, heads or rows too many");
  if (!query || !key || !value || !mask || !out || (count > 0 && (!rows || !pool)))
    return set_error(HS_ERR_INVALID_ARGUMENT, "attend_tree: null pointer");
  TreeParams p{};
  p.batch = batch;
  p.nodes = nodes;
  p.query = query;
  p.key = key;
  p.value = value;
  p.q_batch_stride = query_batch_stride;
  p.q_node_stride = query_node_stride;
  p.kv_batch_stride = kv_batch_stride;
  p.kv_node_stride = kv_node_stride;
  p.mask = mask;
  p.node_counts = node_counts;
  p.pool = pool;
  p.pool_blocks = pool_blocks;
  p.rows = rows;
  p.rows_batch_stride = rows_batch_stride;
  p.count = count;
  p.counts = counts;
  p.out = out;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.head_dim = head_dim;
  p.page_size = page_size;
  p.page_shift = -1;
  if ((page_size & (page_size - 1)) == 0)
    for (int sh = 0; sh < 31; ++sh)
      if ((1 << sh) == page_size) p.page_shift = sh;
  p.groups = q_heads / kv_heads;
  p.splits = tree_splits(batch, nodes, q_heads, kv_heads, count);
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
  const size_t need =
      hs_attend_tree_workspace_bytes(batch, nodes, q_heads, kv_heads, head_dim, count, dtype);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(HS_ERR_WORKSPACE, "attend_tree: workspace of %zu bytes < required %zu",
                     workspace_bytes, need);
  p.partials = static_cast<float *>(workspace);
  p.status = device_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case HS_FLOAT32: return launch<float>(p, s);
    case HS_FLOAT16: return launch<__half>(p, s);
    default: return launch<__nv_bfloat16>(p, s);
  }
}
