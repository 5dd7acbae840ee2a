// (8) Log probabilities of given tokens, entropy and the largest alternatives.
//
// With m the row's maximum, s = sum exp(x - m) and t = sum (x - m) exp(x - m):
// lse = m + log s, the entropy is log s - t / s. Both sums are carried over the
// row with a running maximum: raising it by d scales s by exp(-d) and t to
// exp(-d) (t - d s).
#include <math.h>

#include "common.cuh"
#include "hisparse_verify.h"

namespace hs {
namespace {

constexpr int kLogprobThreads = 256;
constexpr int kLogprobWarps = kLogprobThreads / 32;
constexpr int kMaxTop = 32;

struct LogprobParams {
  const void *logits;
  int64_t row_stride;
  int vocab;
  const void *tokens;
  int tokens64, given;
  float *logprobs, *entropy;
  int top;
  float *top_logprobs;
  int64_t *top_tokens;
  int32_t *status;
};

// Order of an entry as one unsigned word: larger values first, equal values by
// the lower index. NaN ranks above +inf; -0 equals +0.
__device__ __forceinline__ uint32_t value_order(float x) {
  if (x != x) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t entry_order(float x, uint32_t index) {
  return (uint64_t)value_order(x) << 32 | (uint32_t)~index;
}

struct Softmax {
  float m, s, t;
  __device__ __forceinline__ void add(float x) {
    if (x > m || x != x) {  // a new maximum, or NaN, which then stays
      const float d = m - x, f = m == -INFINITY ? 0.f : expf(d);
      t = m == -INFINITY ? 0.f : f * (t + d * s);
      s *= f;
      m = x;
    }
    const float d = x - m, e = m == -INFINITY ? 0.f : expf(d);
    s += e;
    t += e * fmaxf(d, -200.f);  // exp(-200) is 0 in fp32
  }
  __device__ __forceinline__ void join(float m2, float s2, float t2) {
    const float top = m2 > m || m2 != m2 ? m2 : m;
    const float d1 = m - top, d2 = m2 - top;
    const float f1 = m == -INFINITY ? 0.f : expf(d1), f2 = m2 == -INFINITY ? 0.f : expf(d2);
    const float t1 = m == -INFINITY ? 0.f : f1 * (t + d1 * s);
    t = t1 + (m2 == -INFINITY ? 0.f : f2 * (t2 + d2 * s2));
    s = f1 * s + f2 * s2;
    m = top;
  }
};

// One block for each row; the alternatives by one pass over the row for each.
template <typename T>
__global__ void __launch_bounds__(kLogprobThreads) logprobs_kernel(LogprobParams p) {
  __shared__ float sm[kLogprobWarps], ss[kLogprobWarps], st[kLogprobWarps];
  __shared__ uint64_t best[kLogprobWarps];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T *x = static_cast<const T *>(p.logits) + row * p.row_stride;
  Softmax acc{-INFINITY, 0.f, 0.f};
  for (int i = threadIdx.x; i < p.vocab; i += kLogprobThreads) acc.add(to_f32(x[i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    acc.join(__shfl_xor_sync(kFullMask, acc.m, o), __shfl_xor_sync(kFullMask, acc.s, o),
             __shfl_xor_sync(kFullMask, acc.t, o));
  if (lane == 0) {
    sm[warp] = acc.m;
    ss[warp] = acc.s;
    st[warp] = acc.t;
  }
  __syncthreads();
  acc = Softmax{sm[0], ss[0], st[0]};
  for (int w = 1; w < kLogprobWarps; ++w) acc.join(sm[w], ss[w], st[w]);
  const bool empty = acc.m == -INFINITY;
  const float log_s = logf(acc.s);
  // (x - m) - log s: one rounding less than x - lse for entries near the maximum
  auto logprob = [&](float v) { return empty ? -INFINITY : (v - acc.m) - log_s; };
  for (int c = threadIdx.x; c < p.given; c += kLogprobThreads) {
    const int64_t at = row * p.given + c;
    const int64_t token = p.tokens64 ? static_cast<const int64_t *>(p.tokens)[at]
                                     : static_cast<const int32_t *>(p.tokens)[at];
    float v = 0.f;
    if (token >= p.vocab) {
      flag(p.status, HS_DEV_TOKEN_OUT_OF_RANGE);
      v = NAN;
    } else if (token >= 0) {
      v = logprob(to_f32(x[token]));
    }
    p.logprobs[at] = v;
  }
  if (threadIdx.x == 0 && p.entropy != nullptr)
    p.entropy[row] = empty ? 0.f : log_s - acc.t / acc.s;
  uint64_t below = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kLogprobThreads) {
      const uint64_t e = entry_order(to_f32(x[i]), (uint32_t)i);
      if (e < below && e > mine) mine = e;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(kFullMask, mine, o);
      if (other > mine) mine = other;
    }
    __syncthreads();
    if (lane == 0) best[warp] = mine;
    __syncthreads();
    below = best[0];
    for (int w = 1; w < kLogprobWarps; ++w)
      if (best[w] > below) below = best[w];
    if (threadIdx.x == 0) {
      const uint32_t index = ~(uint32_t)below;
      p.top_tokens[row * p.top + k] = index;
      p.top_logprobs[row * p.top + k] = logprob(to_f32(x[index]));
    }
  }
}

template <typename T> int launch(const LogprobParams &p, int64_t rows, cudaStream_t s) {
  logprobs_kernel<T><<<(unsigned)rows, kLogprobThreads, 0, s>>>(p);
  return check_launch("logprobs_kernel");
}

}  // namespace
}  // namespace hs

extern "C" int hs_token_logprobs(int64_t rows, const void *logits, int64_t row_stride, int dtype,
                                 int64_t vocab, const void *tokens, int tokens_dtype, int given,
                                 float *out_logprobs, float *out_entropy, int top,
                                 float *out_top_logprobs, int64_t *out_top_tokens,
                                 int32_t *device_status, hs_stream stream) {
  using namespace hs;
  if (rows < 0 || vocab < 1 || vocab > 0x7fffffff || given < 0 || top < 0 || top > vocab)
    return set_error(HS_ERR_INVALID_ARGUMENT, "logprobs: invalid sizes");
  if (rows > 0x7fffffff) return set_error(HS_ERR_UNSUPPORTED, "logprobs: too many rows");
  if (top > kMaxTop)
    return set_error(HS_ERR_UNSUPPORTED, "logprobs: top %d > %d is not supported", top, kMaxTop);
  if (given > 0 && tokens_dtype != HS_INT32 && tokens_dtype != HS_INT64)
    return set_error(HS_ERR_INVALID_ARGUMENT, "logprobs: tokens must be int32 or int64");
  if (rows == 0) return HS_OK;
  if (!logits || (given > 0 && (!tokens || !out_logprobs)) ||
      (top > 0 && (!out_top_logprobs || !out_top_tokens)))
    return set_error(HS_ERR_INVALID_ARGUMENT, "logprobs: null pointer");
  const LogprobParams p{logits, row_stride, (int)vocab, tokens, tokens_dtype == HS_INT64, given,
                        out_logprobs, out_entropy, top, out_top_logprobs, out_top_tokens,
                        device_status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case HS_FLOAT32: return launch<float>(p, rows, s);
    case HS_FLOAT16: return launch<__half>(p, rows, s);
    case HS_BFLOAT16: return launch<__nv_bfloat16>(p, rows, s);
  }
  return set_error(HS_ERR_INVALID_ARGUMENT, "logprobs: invalid dtype %d", dtype);
}
