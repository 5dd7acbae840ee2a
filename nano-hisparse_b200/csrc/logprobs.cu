// (8) Log probabilities of given tokens, entropy and the largest alternatives.
//
// With m the row's maximum, s = sum exp(x - m) and t = sum (x - m) exp(x - m):
// lse = m + log s, the entropy is log s - t / s. Both sums are carried over the
// row with a running maximum: raising it by d scales s by exp(-d) and t to
// exp(-d) (t - d s). So one pass over the logits gives all of it, and the work is
// bound by reading them once.
//
// The alternatives come out of the same pass: every thread keeps its best entry. At
// least `top` entries of the block's part reach the top-th best of the threads' best
// values, so every one of its `top` largest entries does. Threads whose own best reaches
// it (`top` of them, and equals) have their entries read again for those that do; the
// collected keys are ranked by counting. (A looser bound, the smallest of the warps'
// best, is found in half the time, but made a fifth of the threads read again: half as
// much traffic again on rows that L2 does not hold.)
//
// 2,048 rows of 128,256 take 190 us in fp32 with 5 alternatives (5.5 TB/s, 0.84 of a
// measured copy; 184 us without alternatives, 279 with 32) and 125 us in bf16 (4.2 TB/s;
// 114 without alternatives), bound by about eleven instructions an entry and lane (at 1,184
// rows issue slots 67 % of the cycles, the heavy fp32 pipe 57 %, special functions 49 %, few
// waits for memory). Where more than kCandidates entries of a block pass, the rest of the
// key tells them apart in a second collection (64 rows of equal entries in bf16, 32
// alternatives: 92 us; of random ones 23). Only where the large entries all fall to fewer
// than `top` threads do more than that pass again: those rows take one pass for each
// alternative (307 us).
//
// A row is split over a cluster of 1 to 8 blocks, which join their sums and their
// best keys in the first block's shared memory: few rows reach many SMs without
// a workspace or a second launch.
#include <math.h>

#include "common.cuh"
#include "hisparse_verify.h"

namespace hs {
namespace {

constexpr int kLogprobThreads = 256;  // of a block, or half as many
constexpr int kLogprobWarps = kLogprobThreads / 32;
constexpr int kLogprobBlocks = 4;   // blocks resident on an SM, and twice as many of those
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;
constexpr int kAhead = 4;           // 16-byte vectors in flight per thread
constexpr int kCandidates = 1024;   // keys collected before the exact threshold is taken
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -16384.f;    // exp(kFar) is 0 in fp32

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
  int cluster;
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
__device__ __forceinline__ float order_value(uint64_t order) {
  const uint32_t u = (uint32_t)(order >> 32);
  return u == 0xfffffffeu ? NAN : __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 16 bytes of logits
template <typename T> struct Vector {
  static constexpr int n = 16 / sizeof(T);
  static __device__ __forceinline__ void widen(const uint4 &raw, float (&x)[n]) {
    const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
    for (int i = 0; i < n; ++i) x[i] = to_f32(e[i]);
  }
  static __device__ __forceinline__ float largest(const uint4 &raw) {
    float x[n];
    widen(raw, x);
    float m = x[0];
#pragma unroll
    for (int i = 1; i + 1 < n; i += 2) m = max3_nan(m, x[i], x[i + 1]);
    return max_nan(m, x[n - 1]);
  }
};
// the 16-bit types in pairs
template <typename T2> __device__ __forceinline__ float pair_largest(const uint4 &raw) {
  const T2 *e = reinterpret_cast<const T2 *>(&raw);
  const T2 m = __hmax2_nan(__hmax2_nan(e[0], e[1]), __hmax2_nan(e[2], e[3]));
  return max_nan(to_f32(m.x), to_f32(m.y));
}
template <> __device__ __forceinline__ float Vector<__half>::largest(const uint4 &raw) {
  return pair_largest<__half2>(raw);
}
template <> __device__ __forceinline__ float Vector<__nv_bfloat16>::largest(const uint4 &raw) {
  return pair_largest<__nv_bfloat162>(raw);
}

__device__ __forceinline__ float exp2_flush(float x) {  // below 2^-126: 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Differences are held above kFar where they multiply: a masked entry of -inf or
// of the type's lowest value then adds 0 to t, not 0 * -inf. What that takes from
// NaN and +inf comes back through s, whose own terms stay NaN.
struct Softmax {
  float m, s, t;  // maximum, sum exp(x - m), sum (x - m) exp(x - m)
  __device__ __forceinline__ void raise(float to) {
    if (m != -INFINITY) {
      const float d = fmaxf(m - to, kFar), f = exp2_flush(d * kLog2e);
      t = f * fmaf(d, s, t);
      s *= f;
    }
    m = to;
  }
  __device__ __forceinline__ void add(float x) {  // x <= m
    const float d = x - m, e = exp2_flush(d * kLog2e);
    s += e;
    t = fmaf(e, fmaxf(d, kFar), t);
  }
  // n entries, none above m: two sums of each kind, two products an instruction
  template <int n> __device__ __forceinline__ void add(const float (&x)[n], float2 &s2, float2 &t2) const {
    const float2 below = make_float2(-m, -m), log2e = make_float2(kLog2e, kLog2e);
#pragma unroll
    for (int i = 0; i < n; i += 2) {
      const float2 d = pack_add(make_float2(x[i], x[i + 1]), below), y = pack_mul(d, log2e);
      const float2 e = make_float2(exp2_flush(y.x), exp2_flush(y.y));
      s2 = pack_add(s2, e);
      t2 = pack_fma(e, make_float2(fmaxf(d.x, kFar), fmaxf(d.y, kFar)), t2);
    }
  }
  // the sums over the warp's lanes, in every lane
  __device__ __forceinline__ void join_warp() {
    float top = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(kFullMask, top, o));
    if (m != -INFINITY) {
      const float d = fmaxf(m - top, kFar), f = exp2_flush(d * kLog2e);
      t = f * fmaf(d, s, t);
      s *= f;
    }
    m = top;
    s = warp_xor_tree_sum(s);
    t = warp_xor_tree_sum(t);
  }
  // this lane's part as it was left in shared memory, or none
  __device__ __forceinline__ static Softmax part(const float *from, bool there) {
    return there ? Softmax{from[0], from[1], from[2]} : Softmax{-INFINITY, 0.f, 0.f};
  }
};

__device__ __forceinline__ uint64_t warp_largest(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor_sync(kFullMask, v, o);
    if (other > v) v = other;
  }
  return v;
}

struct LogprobShared {
  float parts[kLogprobWarps][3];  // maximum and sums of each warp
  uint64_t warp_best[kLogprobWarps];
  uint64_t candidates[kCandidates];
  uint64_t best[kMaxTop];
  int found;
  // written by every block of the cluster into the first one's
  float joined[kMaxCluster][3];
  uint64_t joined_best[kMaxCluster * kMaxTop];
};

// The part of a row that a block reads: whole 16-byte vectors, and for the first
// block of a cluster the up to 2 (n - 1) entries before and after them.
template <typename T> struct RowPart {
  static constexpr int n = Vector<T>::n;
  const T *x;
  int head;          // entries before the first vector
  int first, count;  // vectors
  int edge;          // this thread's entry outside the vectors, or -1

  __device__ __forceinline__ RowPart(const LogprobParams &p, const T *row, int rank) : x(row) {
    const int misaligned = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = min(p.vocab, (n - misaligned) % n);
    const int vectors = (p.vocab - head) / n, tail = head + vectors * n;
    const int share = (int)ceil_div(vectors, p.cluster);
    first = min(vectors, rank * share);
    count = min(vectors, first + share) - first;
    const int i = threadIdx.x;
    edge = rank != 0 ? -1 : i < head ? i : i - head < p.vocab - tail ? tail + (i - head) : -1;
  }
  __device__ __forceinline__ uint4 vector(int v) const {
    return __ldg(reinterpret_cast<const uint4 *>(x + head) + first + v);
  }
  __device__ __forceinline__ uint32_t index(int v, int i) const {
    return (uint32_t)(head + (first + v) * n + i);
  }
  // kAhead vectors: v0, v0 + step, ...
  __device__ __forceinline__ void load(int v0, int step, uint4 (&raw)[kAhead]) const {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (v0 + u * step < count) raw[u] = vector(v0 + u * step);
  }
  // f(vector, its number) for vectors v0, v0 + step, ..., kAhead loads at a time
  template <typename F> __device__ __forceinline__ void each(int v0, int step, F f) const {
    for (; v0 < count; v0 += kAhead * step) {
      uint4 raw[kAhead];
      load(v0, step, raw);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (v0 + u * step < count) f(raw[u], v0 + u * step);
    }
  }
};

// Collects the block's entries with a key of at least `threshold`; returns their
// number, of which the first kCandidates are kept. `mine`: a key that no entry of
// this thread passes.
template <int kThreads, typename T>
__device__ __forceinline__ int collect(LogprobShared &sh, const RowPart<T> &part, uint64_t mine,
                                       uint64_t threshold) {
  if (threadIdx.x == 0) sh.found = 0;
  __syncthreads();
  const auto take = [&](uint64_t key) {
    if (key < threshold) return;
    const int at = atomicAdd(&sh.found, 1);
    if (at < kCandidates) sh.candidates[at] = key;
  };
  const uint32_t least = (uint32_t)(threshold >> 32);
  // The whole warp reads the entries of each of its threads that pass, 32 vectors at a
  // time: one thread alone would wait for memory once for every kAhead of them.
  const int lane = threadIdx.x & 31, first = threadIdx.x - lane;
  for (unsigned todo = __ballot_sync(kFullMask, mine >= threshold); todo != 0; todo &= todo - 1) {
    const int owner = first + __ffs(todo) - 1;
    part.each(owner + lane * kThreads, 32 * kThreads, [&](const uint4 &raw, int v) {
      if (value_order(Vector<T>::largest(raw)) < least) return;
      float x[Vector<T>::n];
      Vector<T>::widen(raw, x);
#pragma unroll
      for (int i = 0; i < Vector<T>::n; ++i) take(entry_order(x[i], part.index(v, i)));
    });
  }
  if (mine >= threshold && part.edge >= 0)
    take(entry_order(to_f32(part.x[part.edge]), (uint32_t)part.edge));
  __syncthreads();
  return sh.found;
}

// The block's `top` largest keys into sh.best (0 where it has fewer entries).
// `mine` is this thread's best key, `bound` one that no entry of it passes.
template <int kThreads, typename T>
__device__ __forceinline__ void block_best(LogprobShared &sh, const RowPart<T> &part, int top,
                                           uint64_t mine, uint64_t bound) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < kMaxTop) sh.best[threadIdx.x] = 0;
  // the largest value that the best entries of `top` threads reach, bit by bit
  const auto search = [&](uint64_t known, int from, int to) {
    for (int bit = from; bit >= to; --bit) {
      const uint64_t trial = known | 1ull << bit;
      if (__syncthreads_count(mine >= trial) >= top) known = trial;
    }
    return known;
  };
  // to 16 bits of the value (8 of its fraction in fp32): a few entries more pass than
  // with all of them, for half the steps
  uint64_t threshold = search(0, 63, 48);
  if (threshold == 0) threshold = 1;  // fewer threads with entries than `top`: all of them
  int found = collect<kThreads>(sh, part, bound, threshold);
  if (found > kCandidates) {
    // Many entries are near that value or equal to it: the rest of the key tells them
    // apart, equal ones by their index.
    const uint64_t exact = search(threshold >> 48 << 48, 47, 0);
    if (exact > threshold) {
      threshold = exact;
      found = collect<kThreads>(sh, part, bound, threshold);
    }
  }
  if (found <= kCandidates) {
    for (int i = threadIdx.x; i < found; i += kThreads) {
      const uint64_t key = sh.candidates[i];
      int rank = 0;
      for (int j = 0; j < found; ++j) rank += sh.candidates[j] > key;
      if (rank < top) sh.best[rank] = key;
    }
  } else {  // one pass over the part for each
    uint64_t below = ~0ull;
    for (int k = 0; k < top; ++k) {
      uint64_t next = 0;
      auto take = [&](uint64_t key) {
        if (key < below && key > next) next = key;
      };
      part.each(threadIdx.x, kThreads, [&](const uint4 &raw, int v) {
        float x[Vector<T>::n];
        Vector<T>::widen(raw, x);
#pragma unroll
        for (int i = 0; i < Vector<T>::n; ++i) take(entry_order(x[i], part.index(v, i)));
      });
      if (part.edge >= 0) take(entry_order(to_f32(part.x[part.edge]), (uint32_t)part.edge));
      next = warp_largest(next);
      __syncthreads();
      if (lane == 0) sh.warp_best[warp] = next;
      __syncthreads();
      below = sh.warp_best[0];
      for (int w = 1; w < kThreads / 32; ++w)
        if (sh.warp_best[w] > below) below = sh.warp_best[w];
      if (threadIdx.x == 0) sh.best[k] = below;
    }
  }
  __syncthreads();
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, kLogprobBlocks *kLogprobThreads / kThreads)
    logprobs_kernel(LogprobParams p) {
  constexpr int kWarps = kThreads / 32;
  __shared__ LogprobShared sh;
  const int rank = (int)cluster_rank(), cluster = p.cluster;
  const int64_t row = blockIdx.x / cluster;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // all blocks of the cluster run before any writes to the first one's memory
  if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
  const T *x = static_cast<const T *>(p.logits) + row * p.row_stride;
  const RowPart<T> part(p, x, rank);

  Softmax acc{-INFINITY, 0.f, 0.f};
  int at = -1;  // the vector that first held this thread's maximum
  uint4 raw[kAhead], next[kAhead];
  part.load(threadIdx.x, kThreads, next);
  for (int v0 = threadIdx.x; v0 < part.count; v0 += kAhead * kThreads) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) raw[u] = next[u];
    part.load(v0 + kAhead * kThreads, kThreads, next);  // while these are summed
    float largest = -INFINITY;
    int where = v0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (v0 + u * kThreads < part.count) {
        const float m = Vector<T>::largest(raw[u]);
        if (m > largest || (m != m && largest == largest)) {
          largest = m;
          where = v0 + u * kThreads;
        }
      }
    if (at < 0 || largest > acc.m || (largest != largest && acc.m == acc.m)) {
      at = where;
      acc.raise(largest);
    }
    if (acc.m == -INFINITY) continue;
    float2 s2 = make_float2(acc.s, 0.f), t2 = make_float2(acc.t, 0.f);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (v0 + u * kThreads < part.count) {
        float e[Vector<T>::n];
        Vector<T>::widen(raw[u], e);
        acc.add(e, s2, t2);
      }
    acc.s = s2.x + s2.y;
    acc.t = t2.x + t2.y;
  }
  // This thread's best entry is at most `bound` and at least `mine` in the order:
  // the vector is known, the place in it is not.
  uint64_t mine = 0, bound = 0;
  if (at >= 0) {
    mine = entry_order(acc.m, part.index(at, Vector<T>::n - 1));
    bound = entry_order(acc.m, part.index(at, 0));
  }
  if (part.edge >= 0) {
    const float e = to_f32(x[part.edge]);
    const uint64_t key = entry_order(e, (uint32_t)part.edge);
    if (key > mine) mine = key;
    if (key > bound) bound = key;
    if (e != -INFINITY) {
      if (e > acc.m || e != e) acc.raise(e);
      acc.add(e);
    }
  }
  acc.join_warp();
  if (lane == 0) {
    sh.parts[warp][0] = acc.m;
    sh.parts[warp][1] = acc.s;
    sh.parts[warp][2] = acc.t;
  }
  if (p.top > 0) block_best<kThreads>(sh, part, p.top, mine, bound);
  else __syncthreads();

  if (cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  LogprobShared &out = *(cluster > 1 ? map_rank(&sh, 0) : &sh);
  if (warp == 0) {
    acc = Softmax::part(sh.parts[lane % kWarps], lane < kWarps);
    acc.join_warp();
    if (lane < 3) out.joined[rank][lane] = lane == 0 ? acc.m : lane == 1 ? acc.s : acc.t;
  }
  if (threadIdx.x < p.top) out.joined_best[rank * p.top + threadIdx.x] = sh.best[threadIdx.x];
  if (cluster > 1) {
    cluster_barrier();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  acc = Softmax::part(sh.joined[lane % kMaxCluster], lane < cluster);
  acc.join_warp();
  const bool empty = acc.m == -INFINITY;
  const float log_s = logf(acc.s);
  // (x - m) - log s: one rounding less than x - lse for entries near the maximum
  auto logprob = [&](float v) { return empty ? -INFINITY : (v - acc.m) - log_s; };
  for (int c = threadIdx.x; c < p.given; c += kThreads) {
    const int64_t where = row * p.given + c;
    const int64_t token = p.tokens64 ? static_cast<const int64_t *>(p.tokens)[where]
                                     : static_cast<const int32_t *>(p.tokens)[where];
    float v = 0.f;
    if (token >= p.vocab) {
      flag(p.status, HS_DEV_TOKEN_OUT_OF_RANGE);
      v = NAN;
    } else if (token >= 0) {
      v = logprob(to_f32(x[token]));
    }
    p.logprobs[where] = v;
  }
  if (threadIdx.x == 0 && p.entropy != nullptr)
    p.entropy[row] = empty ? 0.f : log_s - acc.t / acc.s;
  const int keys = cluster * p.top;  // distinct but for the 0 of a block with fewer entries
  if ((int)threadIdx.x < keys) {
    const uint64_t key = sh.joined_best[threadIdx.x];
    int rank_of = 0;
    for (int j = 0; j < keys; ++j) rank_of += sh.joined_best[j] > key;
    if (key != 0 && rank_of < p.top) {
      p.top_tokens[row * p.top + rank_of] = (int64_t)~(uint32_t)key;
      p.top_logprobs[row * p.top + rank_of] = logprob(order_value(key));
    }
  }
}

// Blocks of a row: as many as give every SM's kLogprobBlocks places work, while a
// block still has two rounds of loads to do.
int logprob_cluster(int64_t rows, int64_t row_bytes) {
  const int64_t places = (int64_t)kLogprobBlocks * sm_count();
  const int64_t least = 2 * kAhead * kLogprobThreads * 16;
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= places && row_bytes >= least * c * 2) c *= 2;
  return c;
}

template <typename T> int launch(LogprobParams &p, int64_t rows, cudaStream_t s) {
  static_assert(kMaxCluster * kMaxTop <= kLogprobThreads && kMaxTop <= kLogprobThreads / 2,
                "one thread for each joined key");
  p.cluster = logprob_cluster(rows, (int64_t)p.vocab * sizeof(T));
  if (rows * p.cluster > 0x7fffffff)
    return set_error(HS_ERR_UNSUPPORTED, "logprobs: too many rows");
  // More rows than places: blocks of half the threads, twice as many of them on an SM, let
  // what a block costs besides its reads overlap that of more others. Better for rows of up
  // to 64 KB (2,048 rows of 4,000 in bf16, 5 alternatives: 31 -> 23 us, of 32,000: even) and
  // where it makes one round of two (700 rows of 128,256 in bf16: 66 -> 59); longer rows in
  // more rounds are read faster by large blocks (2,048 of 128,256 in fp32: 204, else 233).
  const int64_t places = (int64_t)kLogprobBlocks * sm_count();
  const bool small = p.cluster == 1 && rows > places &&
                     ((int64_t)p.vocab * sizeof(T) <= 64 * 1024 || rows <= 2 * places);
  const int threads = small ? kLogprobThreads / 2 : kLogprobThreads;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(rows * p.cluster));
  config.blockDim = dim3((unsigned)threads);
  config.stream = s;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = (unsigned)p.cluster;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = p.cluster > 1 ? 1 : 0;
  cudaLaunchKernelEx(&config, threads == kLogprobThreads
                                  ? logprobs_kernel<T, kLogprobThreads>
                                  : logprobs_kernel<T, kLogprobThreads / 2>, p);
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
  LogprobParams p{logits, row_stride, (int)vocab, tokens, tokens_dtype == HS_INT64, given,
                  out_logprobs, out_entropy, top, out_top_logprobs, out_top_tokens,
                  device_status, 1};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case HS_FLOAT32: return launch<float>(p, rows, s);
    case HS_FLOAT16: return launch<__half>(p, rows, s);
    case HS_BFLOAT16: return launch<__nv_bfloat16>(p, rows, s);
  }
  return set_error(HS_ERR_INVALID_ARGUMENT, "logprobs: invalid dtype %d", dtype);
}
