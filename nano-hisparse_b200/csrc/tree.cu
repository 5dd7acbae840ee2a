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
//
// Two kernels: the tensor cores (tree_tensor.cu) serve 16-bit types whose head_dim is a
// multiple of 8 and whose addresses and strides are multiples of 16 bytes; the one below,
// on CUDA cores, everything else. 8 requests of 8 nodes, 8,192 rows, 16 query and 4 KV
// heads of 256 in bf16 take 67 us on the former and 1.6 ms on the latter.
#include "tree.cuh"

namespace hs {
namespace {

// ---- fp32 arithmetic: every type, head_dim and alignment -------------------------------
// 128 threads over a tile of 32 query rows and 32 to 64 keys, operands widened to fp32
// in shared memory. For the scores a thread holds 4 rows x 2 to 4 keys, for the output
// 4 rows x 4 NJ elements, so that four products follow each shared-memory word. A warp
// issues every fifth clock (its products wait for shared memory and for each other), so
// the tile is as small as it takes for two to four blocks on an SM. 8 requests of 8 nodes,
// 2,048 rows, 32 query and 8 KV heads of 128 in fp32: 117 us (131 with 64 keys and two
// blocks, 199 when each tile was loaded after the one before).
constexpr int kSimtThreads = 128;
constexpr int kSimtRows = 32;

template <int NJ> struct SimtShape {
  static constexpr int keys = NJ == 1 ? 64 : NJ == 2 ? 48 : 32;
  static constexpr int resident = NJ == 1 ? 4 : NJ == 2 ? 3 : 2;  // blocks on an SM
  static constexpr int p_pitch = keys + 4;
  static constexpr int dim = 64 * NJ;     // head_dim rounded up
  static constexpr int pitch = dim + 4;   // floats between rows
  static constexpr size_t bytes =
      sizeof(float) * ((kSimtRows + 2 * keys) * pitch + kSimtRows * p_pitch);
  static_assert(resident * (bytes + 1024 + 2048) <= 228 * 1024, "the blocks fit an SM");
};

// Elements d .. d + 3 of a row of head_dim D as fp32, zero past its end. `four`: one
// vector load reads them (D a multiple of 4, addresses of the vector's size).
template <typename T>
__device__ __forceinline__ float4 load_four(const T *row, int d, int D, bool four) {
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (four) {
    if (d < D) load_f32<T, 4>(row + d, x, true);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < D) x[i] = to_f32(row[d + i]);
  }
  return make_float4(x[0], x[1], x[2], x[3]);
}

template <typename T, int NJ>
__global__ void __launch_bounds__(kSimtThreads, SimtShape<NJ>::resident) tree_simt_kernel(TreeParams p, bool four) {
  using Shape = SimtShape<NJ>;
  constexpr int dim = Shape::dim, pitch = Shape::pitch;
  constexpr int keys = Shape::keys, p_pitch = Shape::p_pitch, KJ = keys / 16;
  extern __shared__ __align__(16) float smem[];
  float *sq = smem, *sk = sq + kSimtRows * pitch, *sv = sk + keys * pitch;
  float *sp = sv + keys * pitch;
  // where each key of this tile and the next lives: >= 0 an element offset in the pool,
  // -1 nowhere, -2 - j node j
  __shared__ int64_t s_places[2][keys];
  __shared__ uint64_t s_mask[kSimtRows];
  __shared__ unsigned long long s_bad;  // nodes whose V held a non-finite element
  const int tid = threadIdx.x, split = blockIdx.x;
  const int tiles = (int)ceil_div(p.nodes * p.groups, kSimtRows);
  const int kh = blockIdx.y / tiles, r0 = blockIdx.y % tiles * kSimtRows, b = blockIdx.z;
  const int D = p.head_dim, G = p.groups;
  const int n_nodes = nodes_of(p, b), live = n_nodes * G;  // query rows with a result
  const int64_t valid = rows_of(p, b), total = valid + n_nodes;
  const int64_t chunk = ceil_div(ceil_div(total, p.splits), keys) * keys;
  const int64_t begin = split * chunk, end = min(total, begin + chunk);
  const int tx = tid & 15, ty = tid >> 4;  // keys / elements; rows 4 ty .. 4 ty + 3

  const T *query = static_cast<const T *>(p.query) + b * p.q_batch_stride;
  constexpr int fours = dim / 4;  // a power of two or 48
  for (int i = tid; i < kSimtRows * fours; i += kSimtThreads) {
    const int r = i / fours, d = i % fours * 4, row = r0 + r, t = row / G;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < live)
      x = load_four(query + t * p.q_node_stride + (kh * G + row - t * G) * (int64_t)D, d, D, four);
    *reinterpret_cast<float4 *>(&sq[r * pitch + d]) = x;
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

  const auto look = [&](int64_t k0) -> int64_t {  // the place of key k0 + tid
    const int64_t i = k0 + tid;
    return i >= end ? -1 : i < valid ? row_offset(p, rows[i], row_elems) : -2 - (i - valid);
  };
  // K or V of the keys from k0 on. fp32 rows are copied without registers, but for V
  // of nodes, whose elements that are not finite become 0: nodes that do not see them
  // would meet 0 * NaN. Those that do get them added at the end.
  const auto fill = [&](float *plane, bool values, int64_t k0) {
    const int64_t *places = s_places[(k0 - begin) / keys & 1];
    const bool direct = sizeof(T) == 4 && four && (!values || k0 + keys <= valid);
#pragma unroll 4
    for (int i = tid; i < keys * fours; i += kSimtThreads) {
      const int k = i / fours, d = i % fours * 4;
      const int64_t src = places[k];
      const T *from = src >= 0    ? pool + src + (values ? p.page_size * row_elems : 0)
                      : src < -1 ? (values ? value : key) + (-2 - src) * p.kv_node_stride
                                  : pool;
      float *to = &plane[k * pitch + d];
      if (direct) {
        if (d < D) tree_cp_async16(smem_addr(to), from + d, src != -1);
        continue;
      }
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (src != -1) x = load_four(from, d, D, four);
      if (values && src < -1 &&
          !(fabsf(x.x) < INFINITY && fabsf(x.y) < INFINITY && fabsf(x.z) < INFINITY &&
            fabsf(x.w) < INFINITY)) {
        atomicOr(&s_bad, 1ull << (-2 - src));
        x.x = fabsf(x.x) < INFINITY ? x.x : 0.f;
        x.y = fabsf(x.y) < INFINITY ? x.y : 0.f;
        x.z = fabsf(x.z) < INFINITY ? x.z : 0.f;
        x.w = fabsf(x.w) < INFINITY ? x.w : 0.f;
      }
      *reinterpret_cast<float4 *>(to) = x;
    }
  };
  if (tid == 0) s_bad = 0;
  int64_t ahead = -1;  // the place of key tid of the tile after the next
  if (tid < keys && begin < end) {
    s_places[0][tid] = look(begin);
    ahead = look(begin + keys);
  }
  __syncthreads();
  if (begin < end) fill(sk, false, begin);
  const int used = (D + 3) / 4 * 4;  // elements that are not padding, in fours
  // V of a tile lands while its scores are computed, K of the next one while the output is
  for (int64_t k0 = begin; k0 < end; k0 += keys) {
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    __syncthreads();
    fill(sv, true, k0);
    const int64_t *s_src = s_places[(k0 - begin) / keys & 1];
    if (tid < keys) {
      s_places[((k0 - begin) / keys + 1) & 1][tid] = ahead;
      ahead = look(k0 + 2 * keys);
    }
    float s[4][KJ];  // rows 4 ty + i, keys tx + 16 j
    {
      float2 s2[4][KJ];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < KJ; ++j) s2[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
      for (int d = 0; d < used; d += 4) {
        float4 q4[4], k4[KJ];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q4[i] = *reinterpret_cast<const float4 *>(&sq[(4 * ty + i) * pitch + d]);
#pragma unroll
        for (int j = 0; j < KJ; ++j)
          k4[j] = *reinterpret_cast<const float4 *>(&sk[(tx + 16 * j) * pitch + d]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < KJ; ++j)
            s2[i][j] = pack_fma(make_float2(q4[i].z, q4[i].w), make_float2(k4[j].z, k4[j].w),
                                pack_fma(make_float2(q4[i].x, q4[i].y),
                                         make_float2(k4[j].x, k4[j].y), s2[i][j]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < KJ; ++j) s[i][j] = s2[i][j].x + s2[i][j].y;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
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
      for (int j = 0; j < KJ; ++j) {
        const float w = s[i][j] == -INFINITY ? 0.f : exp2f(s[i][j] - m_new);
        sum += w;
        sp[(4 * ty + i) * p_pitch + tx + 16 * j] = w;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
      l[i] = l[i] * alpha + sum;
      m[i] = m_new;
#pragma unroll
      for (int j = 0; j < 4 * NJ; ++j) acc[i][j] *= alpha;
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    __syncthreads();
    if (k0 + keys < end) fill(sk, false, k0 + keys);
#pragma unroll 2
    for (int k = 0; k < keys; k += 4) {
      float4 w4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w4[i] = *reinterpret_cast<const float4 *>(&sp[(4 * ty + i) * p_pitch + k]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const float4 v4 =
              *reinterpret_cast<const float4 *>(&sv[(k + e) * pitch + 4 * tx + 64 * j]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float w = e == 0 ? w4[i].x : e == 1 ? w4[i].y : e == 2 ? w4[i].z : w4[i].w;
            float *o = &acc[i][4 * j];
            const float2 lo = pack_fma(make_float2(w, w), make_float2(v4.x, v4.y),
                                       make_float2(o[0], o[1]));
            const float2 hi = pack_fma(make_float2(w, w), make_float2(v4.z, v4.w),
                                       make_float2(o[2], o[3]));
            o[0] = lo.x, o[1] = lo.y, o[2] = hi.x, o[3] = hi.y;
          }
        }
    }
  }
  __syncthreads();
  const uint64_t bad = s_bad;
  if (bad != 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t seen = bad & s_mask[4 * ty + i];
#pragma unroll 1
      for (int j = 0; seen != 0 && j < 4 * NJ; ++j) {
        const int d = 4 * tx + 64 * (j / 4) + j % 4;
        const float x = d < D ? nonfinite_sum<T>(p, b, kh, d, seen) : 0.f;
#pragma unroll
        for (int e = 0; e < 4 * NJ; ++e) acc[i][e] += e == j ? x : 0.f;
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
      const int64_t part = part_of(p, b, kh, split);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (4 * tx + 64 * j < D)
          *quad_of(p, part, row, tx + 16 * j) = make_float4(
              acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]);
      if (tx == 0) *stat_of(p, part, row) = make_float2(m[i], l[i]);
    }
  }
}

// ---- joining the splits ------------------------------------------------------------------
// A block joins elements of 8 query rows of a KV head. Warp i takes row i's maxima and
// sums, two splits a lane, to the row's weights exp2(m_s - m); then a thread sums the
// weighted outputs of every kGroups-th split for four neighbouring elements of a row, the
// loads of four splits in flight (the first before the weights are known), and the
// kGroups threads' sums are added through shared memory. With few rows the chain of those
// reads bounds it, so four threads share the splits; with many, or few splits, its
// instructions do, and one thread takes all (4,096 rows of two splits: 2 us of 43 less; 8,192 rows of nine: 4 of 186).
constexpr int kMergeRows = 8, kMergeThreads = 32 * kMergeRows, kMergeAhead = 4;
constexpr int kMergeGroups = 4;

template <typename T, int kGroups>
__global__ void __launch_bounds__(kMergeThreads, 6) tree_merge_kernel(TreeParams p, bool wide) {
  static_assert(kTreeMaxSplits <= 64, "two splits a lane");
  constexpr int kQuads = kMergeThreads / kMergeRows / kGroups, kPlaces = kMergeRows * kQuads;
  __shared__ float weights[kMergeRows][kTreeMaxSplits + 1];  // the last: 1 / sum
  __shared__ float4 sums[kGroups > 1 ? kGroups - 1 : 1][kPlaces];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = p.head_dim;
  const int quads = (D + 3) / 4, slices = (quads + kQuads - 1) / kQuads;
  const int b = blockIdx.z, kh = blockIdx.y, r0 = blockIdx.x / slices * kMergeRows;
  const int all = p.nodes * p.groups, live = nodes_of(p, b) * p.groups;
  const int group = threadIdx.x / kPlaces, place = threadIdx.x % kPlaces;
  const int r = r0 + place % kMergeRows;
  const int quad = blockIdx.x % slices * kQuads + place / kMergeRows;
  const int64_t part = part_of(p, b, kh, 0), step = (int64_t)quads * all;
  const float4 *from = quad_of(p, part, r, quad) + group * step;  // of this thread's first split
  // The splits are written. Every thread waits, also where there is nothing to read:
  // this kernel must not end before the one that writes the workspace.
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  float2 stat[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = lane + 32 * i;
    stat[i] = s < p.splits && r0 + warp < live ? *stat_of(p, part + s, r0 + warp)
                                               : make_float2(-INFINITY, 0.f);
  }
  const bool here = r < live && quad < quads;
  float4 x[kMergeAhead];
  const auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < kMergeAhead; ++i, from += kGroups * step)
      if (here && s0 + i * kGroups < p.splits) x[i] = *from;
  };
  load(group);
  const float m = warp_max(fmaxf(stat[0].x, stat[1].x));
  float weight[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)  // a split that saw nothing left no output: below 0
    weight[i] = stat[i].y == 0.f ? -1.f : tree_exp2(stat[i].x - m);
  const float l = warp_xor_tree_sum(stat[0].y * weight[0] + stat[1].y * weight[1]);
  weights[warp][lane] = weight[0];
  weights[warp][lane + 32] = weight[1];
  if (lane == 0) weights[warp][kTreeMaxSplits] = l > 0.f || l != l ? 1.f / l : 0.f;
  __syncthreads();
  const float *w = weights[place % kMergeRows];
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = group; here && s0 < p.splits; s0 += kMergeAhead * kGroups) {
    if (s0 != group) load(s0);
#pragma unroll
    for (int i = 0; i < kMergeAhead; ++i) {
      const int s = s0 + i * kGroups;
      if (s >= p.splits || w[s] < 0.f) continue;
      sum.x = fmaf(w[s], x[i].x, sum.x);
      sum.y = fmaf(w[s], x[i].y, sum.y);
      sum.z = fmaf(w[s], x[i].z, sum.z);
      sum.w = fmaf(w[s], x[i].w, sum.w);
    }
  }
  if constexpr (kGroups > 1) {
    if (group > 0) sums[group - 1][place] = sum;
    __syncthreads();
  }
  if (group > 0 || r >= all || quad >= quads) return;
#pragma unroll
  for (int g = 0; g < kGroups - 1; ++g) {
    const float4 other = sums[g][place];
    sum = make_float4(sum.x + other.x, sum.y + other.y, sum.z + other.z, sum.w + other.w);
  }
  const float inv = w[kTreeMaxSplits];
  const float y[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
  T *out = static_cast<T *>(p.out) + out_offset(p, b, kh, r) + 4 * quad;
  if constexpr (sizeof(T) == 2) {
    if (wide) {  // rows of whole quads, on 8 bytes
      *reinterpret_cast<uint2 *>(out) = make_uint2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (4 * quad + i < D) out[i] = from_f32<T>(y[i]);
}

template <typename T> int launch_merge(const TreeParams &p, cudaStream_t s) {
  if (p.splits == 1) return HS_OK;
  // threads when one takes all splits of four elements
  const int64_t quads = ceil_div(p.head_dim, 4), rows = (int64_t)p.nodes * p.groups;
  const int64_t threads = quads * rows * p.kv_heads * p.batch;
  const int groups = p.splits > kMergeAhead && threads * kMergeGroups <= (int64_t)2048 * sm_count()
                         ? kMergeGroups : 1;
  const int64_t slices = ceil_div(quads, kMergeThreads / kMergeRows / groups);
  const dim3 grid((unsigned)(ceil_div(rows, kMergeRows) * slices), (unsigned)p.kv_heads,
                  (unsigned)p.batch);
  // its launch overlaps the end of the kernel before it, which it waits for itself
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(kMergeThreads);
  config.stream = s;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  const bool wide = p.head_dim % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
  cudaLaunchKernelEx(&config, groups == 1 ? tree_merge_kernel<T, 1>
                                          : tree_merge_kernel<T, kMergeGroups>, p, wide);
  return check_launch("tree_merge_kernel");
}

// ---- layout of a call ----------------------------------------------------------------------
enum class TreePath { simt, tensor };
// Bytes of `parts` (maximum, sum) pairs before the outputs, which are read and written 16
// bytes at a time.
size_t tree_stats_bytes(size_t parts) { return (parts * sizeof(float2) + 15) / 16 * 16; }

size_t tree_workspace(int64_t rows, int splits, int head_dim) {
  if (splits == 1) return 0;
  const size_t parts = (size_t)rows * splits;
  return tree_stats_bytes(parts) + parts * ((head_dim + 3) / 4) * sizeof(float4);
}

// How a call is laid out: query rows of a block's tile, blocks on an SM, keys of a
// step, splits of the key list.
struct TreeShape {
  TreePath path;
  int rows, resident, keys, splits;
};

TreeShape tree_shape(int batch, int nodes, int q_heads, int kv_heads, int head_dim,
                     int64_t count, int dtype) {
  TreeShape s;
  const int queries = nodes * (q_heads / kv_heads);
  if (dtype == HS_FLOAT32 || head_dim % 8 != 0) {
    s.path = TreePath::simt;
    s.rows = kSimtRows;
    s.resident = head_dim <= 64 ? 4 : head_dim <= 128 ? 3 : 2;
  } else {
    s.path = TreePath::tensor;
    s.rows = 128;
    s.resident = head_dim <= 128 ? 2 : 1;
  }
  s.keys = s.path == TreePath::tensor || head_dim <= 64 ? 64 : head_dim <= 128 ? 48 : 32;
  // The split count with the least (rounds of blocks) x (keys of a block and what a
  // block costs besides, as much as about 384 keys); splits of less than
  // two tiles are not worth joining, but for the fp32 kernel, whose tiles take longest.
  const int64_t blocks = (int64_t)batch * kv_heads * ceil_div(queries, s.rows);
  const int64_t places = (int64_t)s.resident * sm_count(), total = count + nodes;
  int64_t least = 0;
  s.splits = 1;
  for (int n = 1; n <= kTreeMaxSplits; ++n) {
    const int64_t part = ceil_div(ceil_div(total, n), s.keys) * s.keys;
    if (n > 1 && part < (s.path == TreePath::simt ? 1 : 2) * s.keys) break;
    const int64_t cost = ceil_div(blocks * n, places) * (part + 384) + (n > 1 ? 64 : 0);
    if (n == 1 || cost < least) {
      least = cost;
      s.splits = n;
    }
  }
  return s;
}

template <typename T, int NJ> int launch_simt(const TreeParams &p, cudaStream_t s) {
  auto kernel = tree_simt_kernel<T, NJ>;
  const size_t bytes = SimtShape<NJ>::bytes;
  if (int e = reserve_smem(reinterpret_cast<const void *>(kernel), bytes, "attend_tree")) return e;
  const int64_t tiles = ceil_div((int64_t)p.nodes * p.groups, kSimtRows);
  const dim3 grid((unsigned)p.splits, (unsigned)(p.kv_heads * tiles), (unsigned)p.batch);
  // one vector of four elements has an address of its own size
  const uintptr_t addresses =
      reinterpret_cast<uintptr_t>(p.query) | reinterpret_cast<uintptr_t>(p.key) |
      reinterpret_cast<uintptr_t>(p.value) | reinterpret_cast<uintptr_t>(p.pool);
  const int64_t strides =
      p.q_batch_stride | p.q_node_stride | p.kv_batch_stride | p.kv_node_stride;
  const bool four =
      p.head_dim % 4 == 0 && addresses % (4 * sizeof(T)) == 0 && strides % 4 == 0;
  kernel<<<grid, kSimtThreads, bytes, s>>>(p, four);
  return check_launch("tree_simt_kernel");
}

template <typename T>
int launch(const TreeParams &p, TreePath path, int dtype, cudaStream_t s) {
  // the tensor-core kernel copies 16 bytes: every address and stride has to be a multiple,
  // that of the result too where it writes it itself (the join looks at it on its own)
  const uintptr_t addresses =
      reinterpret_cast<uintptr_t>(p.query) | reinterpret_cast<uintptr_t>(p.key) |
      reinterpret_cast<uintptr_t>(p.value) | reinterpret_cast<uintptr_t>(p.pool) |
      (p.splits == 1 ? reinterpret_cast<uintptr_t>(p.out) : 0);
  const int64_t strides =
      p.q_batch_stride | p.q_node_stride | p.kv_batch_stride | p.kv_node_stride;
  if ((addresses & 15) != 0 || (strides & 7) != 0) path = TreePath::simt;
  int status;
  if (path == TreePath::tensor) {
    status = launch_tree_tensor(p, dtype, s);
  } else {
    switch (ceil_div(p.head_dim, 64)) {
      case 1: status = launch_simt<T, 1>(p, s); break;
      case 2: status = launch_simt<T, 2>(p, s); break;
      case 3: status = launch_simt<T, 3>(p, s); break;
      default: status = launch_simt<T, 4>(p, s); break;
    }
  }
  return status != HS_OK ? status : launch_merge<T>(p, s);
}

}  // namespace
}  // namespace hs

extern "C" size_t hs_attend_tree_workspace_bytes(int batch, int nodes, int q_heads, int kv_heads,
                                                 int head_dim, int64_t count, int dtype) {
  using namespace hs;
  if (batch < 1 || nodes < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || count < 0)
    return 0;
  return tree_workspace((int64_t)batch * nodes * q_heads,
                        tree_shape(batch, nodes, q_heads, kv_heads, head_dim, count, dtype).splits,
                        head_dim);
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
  const TreeShape shape = tree_shape(batch, nodes, q_heads, kv_heads, head_dim, count, dtype);
  p.splits = shape.splits;
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
  const size_t need = tree_workspace((int64_t)batch * nodes * q_heads, p.splits, head_dim);
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)
    return set_error(HS_ERR_WORKSPACE, "attend_tree: the workspace must be 16-byte aligned");
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(HS_ERR_WORKSPACE, "attend_tree: workspace of %zu bytes < required %zu",
                     workspace_bytes, need);
  p.stats = static_cast<float2 *>(workspace);
  p.partials = reinterpret_cast<float *>(
      static_cast<char *>(workspace) +
      tree_stats_bytes((size_t)batch * nodes * q_heads * p.splits));
  p.status = device_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case HS_FLOAT32: return launch<float>(p, shape.path, dtype, s);
    case HS_FLOAT16: return launch<__half>(p, shape.path, dtype, s);
    default: return launch<__nv_bfloat16>(p, shape.path, dtype, s);
  }
}
