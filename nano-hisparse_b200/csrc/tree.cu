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

// ---- 16-bit types on the tensor cores ----------------------------------------------------
// 8 warps as kWarpsM x kWarpsN: a warp owns 16 query rows (their fragments of Q
// stay in registers) and 1 / kWarpsN of each stage's keys; warps of the same rows
// join their (O, m, l) at the end. Keys arrive through a ring of kMmaStages
// cp.async stages, 16 bytes a thread, in 16-byte chunks XOR-swizzled by row so
// that ldmatrix meets no bank conflict; the row numbers of a stage are read one
// stage ahead of its copies.
//   S = Q K^T   m16n8k16, K fragments by ldmatrix
//   softmax     fp32 in powers of two; the running maximum is raised only when a
//               score passes it by more than 8 (a factor of 256, far inside
//               fp32 and within fp16's range for P), so O is rescaled rarely
//   O += P V    P rounded to the 16-bit type (a relative error of half a step of
//               each weight, as large as the rounding of the result), V fragments
//               by ldmatrix.trans
// A node's V is copied through registers and its non-finite elements become 0 in
// shared memory: nodes that do not see it would meet 0 * NaN in the product. The
// nodes that do see it get the element added at the end.
constexpr int kMmaThreads = 256;
constexpr int kMmaWarps = kMmaThreads / 32;
constexpr int kMmaStages = 3;
constexpr float kLazy = 8.f;
constexpr unsigned char kPlain = 64, kNothing = 65;  // a key's kind: node 0..63, or these

__device__ __forceinline__ void tree_cp_async16(uint32_t dst, const void *src, bool valid) {
  const int bytes = valid ? 16 : 0;  // 0: zeros are written, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tree_ldmatrix(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tree_ldmatrix_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void tree_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void tree_mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void tree_mma<__half>(float (&c)[4], const uint32_t (&a)[4],
                                                 uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// kDim: head_dim rounded up to the tile (the rest is zero); kWarpsM: 2, 4, 8
template <int kDim, int kWarpsM> struct MmaTile {
  static constexpr int warps_n = kMmaWarps / kWarpsM;
  static constexpr int rows = 16 * kWarpsM;
  static constexpr int stage_keys = 64;
  static constexpr int warp_keys = stage_keys / warps_n;    // 16, 32, 64
  static constexpr int sub_keys = warp_keys < 32 ? warp_keys : 32;
  static constexpr int pitch = kDim * 2;                    // bytes
  static constexpr int stage_bytes = 2 * stage_keys * pitch;
  static constexpr int q_bytes = rows * pitch;
  static constexpr int ring_bytes = kMmaStages * stage_bytes;
  static constexpr int join_pitch = kDim + 4;               // floats
  static constexpr int join_bytes = kMmaWarps * 16 * join_pitch * 4;
  static constexpr size_t bytes =
      q_bytes + (ring_bytes > join_bytes ? ring_bytes : join_bytes) + kMmaStages * stage_keys;
  // blocks on an SM (228 KB, of which every block costs 1 KB besides its own)
  static constexpr int resident = 2 * (bytes + 1280) <= 228 * 1024 ? 2 : 1;
};

template <typename T, int kDim, int kWarpsM>
__global__ void __launch_bounds__(kMmaThreads, (MmaTile<kDim, kWarpsM>::resident))
    tree_mma_kernel(TreeParams p) {
  using Tile = MmaTile<kDim, kWarpsM>;
  constexpr int pitch = Tile::pitch, keys = Tile::stage_keys, chunks = kDim / 8;
  constexpr int row_step = kMmaThreads / chunks, row_loads = keys / row_step;
  constexpr int sub = Tile::sub_keys, nt = sub / 8;  // n-tiles of a sub-tile of scores
  extern __shared__ __align__(128) unsigned char tree_smem[];
  unsigned char *sq = tree_smem, *ring = sq + Tile::q_bytes;
  unsigned char *kinds = tree_smem + Tile::bytes - kMmaStages * keys;
  __shared__ unsigned long long s_bad;  // nodes whose V held a non-finite element
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp % kWarpsM, wn = warp / kWarpsM, split = blockIdx.x;
  const int tiles = (int)ceil_div(p.nodes * p.groups, Tile::rows);
  const int kh = blockIdx.y / tiles, r0 = blockIdx.y % tiles * Tile::rows, b = blockIdx.z;
  const int D = p.head_dim, G = p.groups;
  const int n_nodes = nodes_of(p, b), live = n_nodes * G;
  const int64_t valid = rows_of(p, b);
  const int64_t total = r0 < live ? valid + n_nodes : 0;
  const int64_t chunk = ceil_div(ceil_div(total, p.splits), keys) * keys;
  const int64_t begin = min(total, split * chunk), end = min(total, begin + chunk);
  const int steps = (int)ceil_div(end - begin, keys);
  if (tid == 0) s_bad = 0;

  const int64_t row_elems = (int64_t)p.kv_heads * D;
  const int64_t plane = p.page_size * row_elems;
  const int c = tid % chunks, k_first = tid / chunks;
  const bool in_dim = c * 8 < D;
  const T *pool = static_cast<const T *>(p.pool) + (int64_t)kh * D + c * 8;
  const int64_t node_base = (int64_t)b * p.kv_batch_stride + (int64_t)kh * D + c * 8;
  const T *key = static_cast<const T *>(p.key) + node_base;
  const T *value = static_cast<const T *>(p.value) + node_base;
  const int64_t *rows = p.rows + b * p.rows_batch_stride;

  // the row numbers of a stage's keys that this thread copies a chunk of
  int64_t ahead[row_loads];
  auto look = [&](int step) {
#pragma unroll
    for (int i = 0; i < row_loads; ++i) {
      const int64_t at = begin + (int64_t)step * keys + k_first + i * row_step;
      ahead[i] = at < end && at < valid ? __ldg(rows + at) : -1;
    }
  };
  auto issue = [&](int step) {
    const int slot = step % kMmaStages;
    unsigned char *stage = ring + slot * Tile::stage_bytes;
#pragma unroll
    for (int i = 0; i < row_loads; ++i) {
      const int k = k_first + i * row_step;
      const int64_t at = begin + (int64_t)step * keys + k;
      const uint32_t place = k * pitch + ((c ^ (k & 7)) << 4);
      if (at >= valid && at < end) {  // a node
        const int j = (int)(at - valid);
        uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
        if (in_dim) {
          kx = *reinterpret_cast<const uint4 *>(key + j * p.kv_node_stride);
          vx = *reinterpret_cast<const uint4 *>(value + j * p.kv_node_stride);
        }
        T *v = reinterpret_cast<T *>(&vx);
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!(fabsf(to_f32(v[e])) < INFINITY)) {
            v[e] = from_f32<T>(0.f);
            bad = true;
          }
        if (bad) atomicOr(&s_bad, 1ull << j);
        *reinterpret_cast<uint4 *>(stage + place) = kx;
        *reinterpret_cast<uint4 *>(stage + keys * pitch + place) = vx;
        if (c == 0) kinds[slot * keys + k] = (unsigned char)j;
      } else {
        const int64_t off = row_offset(p, ahead[i], row_elems);
        const bool ok = off >= 0;
        const T *src = ok ? pool + off : pool;
        tree_cp_async16(smem_addr(stage + place), src, ok && in_dim);
        tree_cp_async16(smem_addr(stage + keys * pitch + place), ok ? src + plane : src,
                        ok && in_dim);
        if (c == 0) kinds[slot * keys + k] = ok ? kPlain : kNothing;
      }
    }
  };
  if (steps > 0) look(0);
  __syncthreads();  // s_bad
#pragma unroll
  for (int s = 0; s < kMmaStages - 1; ++s) {
    if (s < steps) {
      issue(s);
      look(s + 1);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  }

  // Q: rows r0 .., zero beyond the last
  const T *query = static_cast<const T *>(p.query) + b * p.q_batch_stride;
  for (int i = tid; i < Tile::rows * chunks; i += kMmaThreads) {
    const int r = i / chunks, qc = i % chunks, row = r0 + r;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (row < live && qc * 8 < D)
      x = *reinterpret_cast<const uint4 *>(query + row / G * p.q_node_stride +
                                           (int64_t)(kh * G + row % G) * D + qc * 8);
    *reinterpret_cast<uint4 *>(sq + r * pitch + ((qc ^ (r & 7)) << 4)) = x;
  }
  __syncthreads();
  // lane's two rows, and what their nodes see
  const int row_lo = r0 + wm * 16 + lane / 4, row_hi = row_lo + 8;
  uint64_t see_lo = 0, see_hi = 0;
  if (row_lo < live) see_lo = (uint64_t)p.mask[(int64_t)b * p.nodes + row_lo / G];
  if (row_hi < live) see_hi = (uint64_t)p.mask[(int64_t)b * p.nodes + row_hi / G];

  constexpr bool q_in_registers = kDim <= 128;
  uint32_t qf[q_in_registers ? kDim / 16 : 1][4];
  const int q_row = wm * 16 + (lane & 15);
  auto load_q = [&](int kk, uint32_t (&f)[4]) {
    tree_ldmatrix(smem_addr(sq + q_row * pitch + (((2 * kk + (lane >> 4)) ^ (q_row & 7)) << 4)),
                  f);
  };
  if constexpr (q_in_registers)
#pragma unroll
    for (int kk = 0; kk < kDim / 16; ++kk) load_q(kk, qf[kk]);

  float o[kDim / 8][4];
#pragma unroll
  for (int j = 0; j < kDim / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
  float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;

  for (int step = 0; step < steps; ++step) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kMmaStages - 2) : "memory");
    __syncthreads();
    if (step + kMmaStages - 1 < steps) {
      issue(step + kMmaStages - 1);
      look(step + kMmaStages);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    const int slot = step % kMmaStages;
    const unsigned char *sk = ring + slot * Tile::stage_bytes, *sv = sk + keys * pitch;
#pragma unroll
    for (int part = 0; part < Tile::warp_keys / sub; ++part) {
      const int k0 = wn * Tile::warp_keys + part * sub;
      float s[nt][4];
#pragma unroll
      for (int j = 0; j < nt; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < kDim / 16; ++kk) {
        uint32_t af[4];
        if constexpr (q_in_registers) {
#pragma unroll
          for (int e = 0; e < 4; ++e) af[e] = qf[kk][e];
        } else {
          load_q(kk, af);
        }
#pragma unroll
        for (int j = 0; j < nt; j += 2) {
          // keys 8 j .. 8 j + 15: lanes 0-7 rows 0-7 low half, 8-15 its high half, then rows 8-15
          const int kr = k0 + j * 8 + (lane & 7) + ((lane >> 4) << 3);
          const int kc = 2 * kk + ((lane >> 3) & 1);
          uint32_t kf[4];
          tree_ldmatrix(smem_addr(sk + kr * pitch + ((kc ^ (kr & 7)) << 4)), kf);
          tree_mma<T>(s[j], af, kf[0], kf[1]);
          tree_mma<T>(s[j + 1], af, kf[2], kf[3]);
        }
      }
      // what each score's key is: two keys a 16-bit word
      bool plain = true;
      unsigned kind[nt];
#pragma unroll
      for (int j = 0; j < nt; ++j) {
        kind[j] = *reinterpret_cast<const unsigned short *>(
            kinds + slot * keys + k0 + j * 8 + (lane & 3) * 2);
        plain = plain && kind[j] == (kPlain | kPlain << 8);
      }
      float top_lo = -INFINITY, top_hi = -INFINITY;
#pragma unroll
      for (int j = 0; j < nt; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] *= p.scale_log2;
        if (!plain) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const unsigned kd = kind[j] >> (8 * e) & 0xff;
            if (kd == kNothing || (kd < kPlain && !(see_lo >> kd & 1))) s[j][e] = -INFINITY;
            if (kd == kNothing || (kd < kPlain && !(see_hi >> kd & 1))) s[j][2 + e] = -INFINITY;
          }
        }
        top_lo = fmaxf(top_lo, fmaxf(s[j][0], s[j][1]));
        top_hi = fmaxf(top_hi, fmaxf(s[j][2], s[j][3]));
      }
      const bool raise = top_lo > m_lo + kLazy || top_hi > m_hi + kLazy;
      if (__any_sync(kFullMask, raise)) {
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {
          top_lo = fmaxf(top_lo, __shfl_xor_sync(kFullMask, top_lo, d));
          top_hi = fmaxf(top_hi, __shfl_xor_sync(kFullMask, top_hi, d));
        }
        const float new_lo = fmaxf(m_lo, top_lo), new_hi = fmaxf(m_hi, top_hi);
        const float f_lo = m_lo == -INFINITY ? 0.f : exp2_fast(m_lo - new_lo);
        const float f_hi = m_hi == -INFINITY ? 0.f : exp2_fast(m_hi - new_hi);
        m_lo = new_lo;
        m_hi = new_hi;
        l_lo *= f_lo;
        l_hi *= f_hi;
#pragma unroll
        for (int j = 0; j < kDim / 8; ++j) {
          o[j][0] *= f_lo;
          o[j][1] *= f_lo;
          o[j][2] *= f_hi;
          o[j][3] *= f_hi;
        }
      }
      // a row that has seen nothing keeps m = -inf: its weights are exp2(-inf) = 0
      const float b_lo = m_lo == -INFINITY ? 0.f : m_lo, b_hi = m_hi == -INFINITY ? 0.f : m_hi;
#pragma unroll
      for (int j = 0; j < nt; ++j) {
        s[j][0] = exp2_fast(s[j][0] - b_lo);
        s[j][1] = exp2_fast(s[j][1] - b_lo);
        s[j][2] = exp2_fast(s[j][2] - b_hi);
        s[j][3] = exp2_fast(s[j][3] - b_hi);
        l_lo += s[j][0] + s[j][1];
        l_hi += s[j][2] + s[j][3];
      }
#pragma unroll
      for (int kk = 0; kk < sub / 16; ++kk) {
        const uint32_t pf[4] = {pack2<T>(s[2 * kk][0], s[2 * kk][1]),
                                pack2<T>(s[2 * kk][2], s[2 * kk][3]),
                                pack2<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                                pack2<T>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
        const int vr = k0 + kk * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < kDim / 8; j += 2) {
          uint32_t vf[4];
          tree_ldmatrix_trans(
              smem_addr(sv + vr * pitch + (((j + (lane >> 4)) ^ (vr & 7)) << 4)), vf);
          tree_mma<T>(o[j], pf, vf[0], vf[1]);
          tree_mma<T>(o[j + 1], pf, vf[2], vf[3]);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
  for (int d = 1; d <= 2; d <<= 1) {
    l_lo += __shfl_xor_sync(kFullMask, l_lo, d);
    l_hi += __shfl_xor_sync(kFullMask, l_hi, d);
  }
  // join the warps of the same rows through the ring's memory
  __syncthreads();
  float *join = reinterpret_cast<float *>(ring);
  constexpr int jp = Tile::join_pitch;
  {
    float *lo = join + (warp * 16 + lane / 4) * jp, *hi = lo + 8 * jp;
#pragma unroll
    for (int j = 0; j < kDim / 8; ++j) {
      const int d = j * 8 + (lane & 3) * 2;
      *reinterpret_cast<float2 *>(lo + d) = make_float2(o[j][0], o[j][1]);
      *reinterpret_cast<float2 *>(hi + d) = make_float2(o[j][2], o[j][3]);
    }
    if ((lane & 3) == 0) {
      lo[kDim] = m_lo;
      lo[kDim + 1] = l_lo;
      hi[kDim] = m_hi;
      hi[kDim + 1] = l_hi;
    }
  }
  __syncthreads();
  const unsigned long long bad = s_bad;
  T *out = static_cast<T *>(p.out) + (int64_t)b * p.nodes * p.q_heads * D;
  const int rows_here = min(Tile::rows, p.nodes * G - r0);
  for (int r = warp; r < rows_here; r += kMmaWarps) {
    const int row = r0 + r;
    const float *first = join + (r / 16 * 16 + r % 16) * jp;  // warp r / 16 of column wn = 0
    float m = -INFINITY, l = 0.f, w[Tile::warps_n];
#pragma unroll
    for (int k = 0; k < Tile::warps_n; ++k) m = fmaxf(m, first[k * kWarpsM * 16 * jp + kDim]);
#pragma unroll
    for (int k = 0; k < Tile::warps_n; ++k) {
      const float mk = first[k * kWarpsM * 16 * jp + kDim];
      w[k] = mk == -INFINITY ? 0.f : exp2_fast(mk - m);
      l += first[k * kWarpsM * 16 * jp + kDim + 1] * (mk == -INFINITY ? 1.f : w[k]);
    }
    const uint64_t see = bad != 0 && row < live ? (uint64_t)p.mask[(int64_t)b * p.nodes + row / G] : 0;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    for (int d = lane; d < D; d += 32) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < Tile::warps_n; ++k) x = fmaf(first[k * kWarpsM * 16 * jp + d], w[k], x);
      for (uint64_t todo = bad & see; todo != 0; todo &= todo - 1) {
        const int j = __ffsll((long long)todo) - 1;
        const float v = to_f32(static_cast<const T *>(p.value)[(int64_t)b * p.kv_batch_stride +
                                                               j * p.kv_node_stride +
                                                               (int64_t)kh * D + d]);
        if (!(fabsf(v) < INFINITY)) x += v;
      }
      if (p.splits == 1)
        out[(int64_t)(row / G) * p.q_heads * D + (int64_t)(kh * G + row % G) * D + d] =
            from_f32<T>(row < live ? x * inv : 0.f);
      else
        partial_of(p, b, kh, row, split)[d] = x;
    }
    if (p.splits > 1 && lane == 0) {
      float *part = partial_of(p, b, kh, row, split);
      part[D] = m;
      part[D + 1] = l;
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

// How a call is laid out: query rows of a block's tile, blocks on an SM, keys of a
// step, splits of the key list.
struct TreeShape {
  int rows, resident, keys, splits;
  bool mma;
};

TreeShape tree_shape(int batch, int nodes, int q_heads, int kv_heads, int head_dim,
                     int64_t count, int dtype) {
  TreeShape s;
  const int queries = nodes * (q_heads / kv_heads);
  s.mma = dtype != HS_FLOAT32 && head_dim % 8 == 0;
  if (s.mma) {
    s.rows = queries <= 32 ? 32 : queries <= 64 || head_dim > 128 ? 64 : 128;
    s.keys = 64;
    s.resident = head_dim <= 64 || (head_dim <= 128 && s.rows <= 64) ? 2 : 1;
  } else {
    s.rows = kSimtRows;
    s.keys = kSimtKeys;
    s.resident = 2;
  }
  // The split count with the least (rounds of blocks) x (keys of a block and what a
  // block costs besides, about 128 keys); more splits than two tiles each are not
  // worth joining.
  const int64_t blocks = (int64_t)batch * kv_heads * ceil_div(queries, s.rows);
  const int64_t places = (int64_t)s.resident * sm_count(), total = count + nodes;
  int64_t least = 0;
  s.splits = 1;
  for (int n = 1; n <= kTreeMaxSplits; ++n) {
    const int64_t part = ceil_div(ceil_div(total, n), s.keys) * s.keys;
    if (n > 1 && part < 2 * s.keys) break;
    const int64_t cost = ceil_div(blocks * n, places) * (part + 128) + (n > 1 ? 64 : 0);
    if (n == 1 || cost < least) {
      least = cost;
      s.splits = n;
    }
  }
  return s;
}

template <typename T> int launch_merge(const TreeParams &p, cudaStream_t s) {
  if (p.splits == 1) return HS_OK;
  const dim3 merge((unsigned)p.nodes, (unsigned)p.q_heads, (unsigned)p.batch);
  tree_merge_kernel<T><<<merge, (unsigned)(ceil_div(p.head_dim, 32) * 32), 0, s>>>(p);
  return check_launch("tree_merge_kernel");
}

template <typename T, int NJ> int launch_simt(const TreeParams &p, cudaStream_t s) {
  auto kernel = tree_simt_kernel<T, NJ>;
  const size_t bytes = SimtShape<NJ>::bytes;
  if (int e = reserve_smem(reinterpret_cast<const void *>(kernel), bytes, "attend_tree")) return e;
  const int64_t tiles = ceil_div((int64_t)p.nodes * p.groups, kSimtRows);
  const dim3 grid((unsigned)p.splits, (unsigned)(p.kv_heads * tiles), (unsigned)p.batch);
  kernel<<<grid, kSimtThreads, bytes, s>>>(p);
  if (int e = check_launch("tree_simt_kernel")) return e;
  return launch_merge<T>(p, s);
}

template <typename T, int kDim, int kWarpsM> int launch_mma(const TreeParams &p, cudaStream_t s) {
  using Tile = MmaTile<kDim, kWarpsM>;
  auto kernel = tree_mma_kernel<T, kDim, kWarpsM>;
  if (int e = reserve_smem(reinterpret_cast<const void *>(kernel), Tile::bytes, "attend_tree"))
    return e;
  const int64_t tiles = ceil_div((int64_t)p.nodes * p.groups, Tile::rows);
  const dim3 grid((unsigned)p.splits, (unsigned)(p.kv_heads * tiles), (unsigned)p.batch);
  kernel<<<grid, kMmaThreads, Tile::bytes, s>>>(p);
  if (int e = check_launch("tree_mma_kernel")) return e;
  return launch_merge<T>(p, s);
}

template <typename T, int kDim>
int launch_rows(const TreeParams &p, const TreeShape &shape, cudaStream_t s) {
  if (shape.rows == 32) return launch_mma<T, kDim, 2>(p, s);
  if constexpr (kDim <= 128)  // 128 rows of Q and the ring pass an SM's memory at 256
    if (shape.rows == 128) return launch_mma<T, kDim, 8>(p, s);
  return launch_mma<T, kDim, 4>(p, s);
}

template <typename T> int launch(const TreeParams &p, const TreeShape &shape, cudaStream_t s) {
  // the copies are 16 bytes: every address and stride has to be a multiple
  const uintptr_t addresses =
      reinterpret_cast<uintptr_t>(p.query) | reinterpret_cast<uintptr_t>(p.key) |
      reinterpret_cast<uintptr_t>(p.value) | reinterpret_cast<uintptr_t>(p.pool);
  const int64_t strides =
      p.q_batch_stride | p.q_node_stride | p.kv_batch_stride | p.kv_node_stride;
  if constexpr (sizeof(T) == 2)
    if (shape.mma && (addresses & 15) == 0 && (strides & 7) == 0) {
      if (p.head_dim <= 64) return launch_rows<T, 64>(p, shape, s);
      if (p.head_dim <= 128) return launch_rows<T, 128>(p, shape, s);
      return launch_rows<T, 256>(p, shape, s);
    }
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
  if (batch < 1 || nodes < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || count < 0)
    return 0;
  const int splits =
      tree_shape(batch, nodes, q_heads, kv_heads, head_dim, count, dtype).splits;
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
  const TreeShape shape = tree_shape(batch, nodes, q_heads, kv_heads, head_dim, count, dtype);
  p.splits = shape.splits;
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
    case HS_FLOAT32: return launch<float>(p, shape, s);
    case HS_FLOAT16: return launch<__half>(p, shape, s);
    default: return launch<__nv_bfloat16>(p, shape, s);
  }
}
