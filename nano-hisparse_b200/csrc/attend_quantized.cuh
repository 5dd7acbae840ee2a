// What the attention kernels over an 8-bit cache share; attend_quantized.cu has the
// formulas and the entry points.
#pragma once

#include <math.h>

#include "quantized.cuh"

namespace hs {

constexpr int kQuantMaxSplits = 128;
constexpr int kClusterSplits = 8;  // joined in the kernel, as a cluster
constexpr float kSumLift = 10.f, kSumScale = 1024.f;  // 2^kSumLift

struct QuantAttendParams {
  int batch;
  const void *query;
  int64_t q_batch_stride;
  const unsigned char *pool;
  int64_t pool_blocks, record;
  const int64_t *rows;
  int64_t rows_batch_stride, rows_head_stride, count;
  const int32_t *counts32;  // rows of a request: counts32, or the sum of counts64, or `count`
  const int64_t *counts64;
  int counts_stride, counts_first, counts_n;
  void *out;            // written where no other kernel joins the splits, else NULL
  int q_heads, kv_heads, head_dim, page_size, page_shift;
  int groups;           // query heads of a KV head
  int splits, phase;
  bool join;            // the splits' results go by way of the workspace
  float scale_log2;     // log2(e) / sqrt(head_dim): scores are kept in powers of two
  // [phases][batch][q_heads][splits]: the maximum's score and V exponent, the sum; and
  // [.. , quads of 4] outputs
  float4 *stats;
  float *partials;
  int32_t *status;
};

__device__ __forceinline__ int64_t quant_rows(const QuantAttendParams &p, int b) {
  int64_t n = p.count;
  if (p.counts32 != nullptr) {
    n = p.counts32[b];
  } else if (p.counts64 != nullptr) {
    n = 0;
    for (int i = 0; i < p.counts_n; ++i)
      n += p.counts64[(int64_t)b * p.counts_stride + p.counts_first + i];
  }
  return n < 0 ? 0 : (n > p.count ? p.count : n);
}
__host__ __device__ __forceinline__ int quant_pad(int head_dim) { return (head_dim + 3) / 4 * 4; }
// Index of a partial result
__device__ __forceinline__ int64_t quant_part(const QuantAttendParams &p, int phase, int b, int h,
                                              int split) {
  return (((int64_t)phase * p.batch + b) * p.q_heads + h) * p.splits + split;
}
__device__ __forceinline__ float quant_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The partial result with the larger maximum; one that saw nothing has sum 0, and one
// whose sum is NaN counts as the largest.
__device__ __forceinline__ float4 quant_larger(float4 a, float4 b) {
  if (a.z == 0.f || b.z != b.z) return b;
  if (b.z == 0.f || a.z != a.z) return a;
  return b.x + b.y > a.x + a.y ? b : a;
}
// 2^(s + e) over 2^(top_s + top_e), e and top_e whole: adding them last keeps the scores'
// difference exact where scores are near each other and exponents are large.
__device__ __forceinline__ float quant_share(float s, float e, float top_s, float top_e) {
  return quant_exp2((s - top_s) + (e - top_e));
}

// attend_quantized_mma.cu: head_dim a multiple of 16, shared rows, query and its stride
// multiples of four elements, fewer than 2^32 records
// It joins up to kClusterSplits splits itself where p.out is given.
struct QuantMmaGrid {
  int queries, chunks;         // query heads of a warp, such parts of a KV head's
  int heads, groups, places;   // KV heads of a block, such blocks, warps side by side
  int slices;                  // warps that share a head's rows
  int resident;                // blocks on an SM
};
QuantMmaGrid quant_mma_grid(int dtype, int q_heads, int kv_heads, int head_dim);
int launch_quant_mma(const QuantAttendParams &p, int dtype, cudaStream_t s);

}  // namespace hs
