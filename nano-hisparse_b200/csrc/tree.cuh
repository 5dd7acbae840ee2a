// What the tree attention kernels share; tree.cu has the formulas and the entry point.
#pragma once

#include <math.h>

#include "common.cuh"
#include "hisparse_verify.h"

namespace hs {

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
  // unnormalised outputs, four elements of a row together:
  // [batch][kv_heads][splits][ceil(head_dim / 4)][nodes * groups][4]
  float *partials;
  float2 *stats;        // [batch][kv_heads][splits][nodes * groups]: maximum, sum
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

// What a split leaves: (maximum, sum) of query row r is stat_of(...), elements
// 4 i .. 4 i + 3 of its unnormalised output are quad_of(..., i). The threads of the
// tcgen05 kernel and of the joining one have a row each: theirs are neighbours.
__device__ __forceinline__ int64_t part_of(const TreeParams &p, int b, int kh, int split) {
  return ((int64_t)b * p.kv_heads + kh) * p.splits + split;
}
__device__ __forceinline__ float2 *stat_of(const TreeParams &p, int64_t part, int r) {
  return p.stats + part * (p.nodes * p.groups) + r;
}
__device__ __forceinline__ float4 *quad_of(const TreeParams &p, int64_t part, int r, int i) {
  return reinterpret_cast<float4 *>(p.partials) +
         (part * ((p.head_dim + 3) / 4) + i) * (p.nodes * p.groups) + r;
}

// Where query row r of KV head kh starts in the output.
__device__ __forceinline__ int64_t out_offset(const TreeParams &p, int b, int kh, int r) {
  const int t = r / p.groups;
  return (((int64_t)b * p.nodes + t) * p.q_heads + kh * p.groups + r - t * p.groups) * p.head_dim;
}

__device__ __forceinline__ float tree_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
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

__device__ __forceinline__ void tree_cp_async16(uint32_t dst, const void *src, bool valid) {
  const int bytes = valid ? 16 : 0;  // 0: zeros are written, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}

// A weight is kept as 2^(score - maximum + kLift): with the maximum raised only
// past kLazy, fp16 weights stay below 2^15 and their smallest normal is 2^-21.
constexpr float kLazy = 8.f;
template <typename T> constexpr float kLift = 0.f;
template <> constexpr float kLift<__half> = 7.f;

// A node's V element that is not finite becomes 0 in shared memory: nodes that do
// not see it would meet 0 * NaN in the product. Returns whether there was one.
template <typename T> __device__ __forceinline__ bool clear_nonfinite(uint4 &raw) {
  T *v = reinterpret_cast<T *>(&raw);
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (!(fabsf(to_f32(v[e])) < INFINITY)) {
      v[e] = from_f32<T>(0.f);
      bad = true;
    }
  return bad;
}
// What those elements add to element d of a row that sees the nodes `seen`: the
// result is not finite either way, so their weights do not matter.
template <typename T>
__device__ __forceinline__ float nonfinite_sum(const TreeParams &p, int b, int kh, int d,
                                               uint64_t seen) {
  float x = 0.f;
  for (; seen != 0; seen &= seen - 1) {
    const int j = __ffsll((long long)seen) - 1;
    const float v = to_f32(static_cast<const T *>(
        p.value)[(int64_t)b * p.kv_batch_stride + j * p.kv_node_stride +
                 (int64_t)kh * p.head_dim + d]);
    if (!(fabsf(v) < INFINITY)) x += v;
  }
  return x;
}

// tree_tensor.cu: 16-bit types, head_dim a multiple of 8
int launch_tree_tensor(const TreeParams &p, int dtype, cudaStream_t s);

}  // namespace hs
