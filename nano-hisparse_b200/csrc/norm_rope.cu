// (6) Per-head RMS norms of queries and keys with the position rotation.
//
// y = x / sqrt(mean(x^2) + eps) * w, then the pair (y_i, y_{i+R}) turns by the
// angle positions[n] * inv_freq[i], R = head_dim / 2. Every element is read and
// written once; the sums, the norm and the rotation are fp32 and the result is
// rounded to the element type once.
//
// The angle: a position of one million times an inverse frequency of 1 is
// 159,155 turns; fp32 would keep the angle to 0.03 rad only. The product is
// formed in fp64 in units of a turn, its whole turns are dropped there, and
// sincospif() takes the remaining fraction in fp32 (an error of at most
// 2^-25 turn, 1.9e-7 rad).
//
// Bound by HBM: 32,768 tokens of 40 heads of 128 in bf16 take 126 us, 5.3 TB/s (0.81 of
// a measured copy); one token 2.2 us. The kernel of 16-byte vectors serves
// aligned inputs, the other one every even head_dim, stride and address (463 us there).
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "hisparse_verify.h"

namespace hs {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeWarps = kRopeThreads / 32;
constexpr int kRopeMaxDim = 256;
constexpr int kRopeResident = 3;  // blocks on an SM

struct RopeParams {
  int64_t tokens;
  const void *in[2];  // query, key
  int64_t token_stride[2], head_stride[2];
  int heads[2];
  const void *weight[2];
  void *out[2];
  int head_dim;
  const void *positions;
  int positions64;
  const double *inv_freq;
  float eps;
};

__device__ __forceinline__ double position_of(const RopeParams &p, int64_t n) {
  return p.positions64 ? (double)static_cast<const int64_t *>(p.positions)[n]
                       : (double)static_cast<const int32_t *>(p.positions)[n];
}

// cos and sin of position * inv_freq
__device__ __forceinline__ void turn(double position, double inv_freq, float &cosine,
                                     float &sine) {
  constexpr double kInvTwoPi = 0.15915494309189533577;
  const double turns = position * inv_freq * kInvTwoPi;
  sincospif(2.f * (float)(turns - rint(turns)), &sine, &cosine);
}

// One warp for each (token, head); lane l holds the pairs l, l + 32, ... Serves
// every even head_dim, stride and alignment.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) norm_rope_any_kernel(RopeParams p) {
  constexpr int kPairs = kRopeMaxDim / 2 / 32;
  const int lane = threadIdx.x & 31;
  const int all = p.heads[0] + p.heads[1];
  const int64_t item = (int64_t)blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
  if (item >= p.tokens * all) return;
  const int64_t n = item / all;
  int h = (int)(item % all);
  const int which = h >= p.heads[0];
  if (which) h -= p.heads[0];
  const int half = p.head_dim / 2;
  const T *x = static_cast<const T *>(p.in[which]) + n * p.token_stride[which] +
               h * p.head_stride[which];
  float a[kPairs], b[kPairs], sum = 0.f;
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const int i = lane + 32 * j;
    a[j] = i < half ? to_f32(x[i]) : 0.f;
    b[j] = i < half ? to_f32(x[i + half]) : 0.f;
    sum = fmaf(a[j], a[j], fmaf(b[j], b[j], sum));
  }
  const T *w = static_cast<const T *>(p.weight[which]);
  float scale = 1.f;
  if (w != nullptr) scale = rsqrtf(warp_xor_tree_sum(sum) / (float)p.head_dim + p.eps);
  const double position = position_of(p, n);
  T *out = static_cast<T *>(p.out[which]) + (n * p.heads[which] + h) * p.head_dim;
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const int i = lane + 32 * j;
    if (i >= half) break;
    float cosine, sine;
    turn(position, p.inv_freq[i], cosine, sine);
    const float ya = a[j] * scale * (w ? to_f32(w[i]) : 1.f);
    const float yb = b[j] * scale * (w ? to_f32(w[i + half]) : 1.f);
    out[i] = from_f32<T>(ya * cosine - yb * sine);
    out[i + half] = from_f32<T>(yb * cosine + ya * sine);
  }
}

// The same with 16-byte loads: lane j of a group of kGroup lanes holds the pairs
// j * kVec .. of one head, a warp 32 / kGroup heads at once. A warp walks `span`
// head sets of one token with the lane's cosines and sines in registers; a set's loads
// are issued before the set before it is worked on, the first before the angles. Products
// are packed, two fp32 an instruction: a plain copy in this form takes 111 us at 32,768
// tokens of 40 heads, so the instructions are what costs beyond the bytes.
template <typename T, int kPairs>  // 16 bytes as pairs of fp32
__device__ __forceinline__ void unpack(const uint4 &raw, float2 (&x)[kPairs]) {
  const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) x[i] = make_float2(to_f32(e[2 * i]), to_f32(e[2 * i + 1]));
}
template <typename T, int kPairs>
__device__ __forceinline__ uint4 pack(const float2 (&x)[kPairs]) {
  uint4 raw;
  uint32_t *words = reinterpret_cast<uint32_t *>(&raw);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    if constexpr (sizeof(T) == 4) {
      words[2 * i] = __float_as_uint(x[i].x);
      words[2 * i + 1] = __float_as_uint(x[i].y);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 v = __floats2half2_rn(x[i].x, x[i].y);
      words[i] = *reinterpret_cast<const uint32_t *>(&v);
    } else {
      const __nv_bfloat162 v = __floats2bfloat162_rn(x[i].x, x[i].y);
      words[i] = *reinterpret_cast<const uint32_t *>(&v);
    }
  }
  return raw;
}

__device__ __forceinline__ uint4 choose(bool first, const uint4 &a, const uint4 &b) {
  return make_uint4(first ? a.x : b.x, first ? a.y : b.y, first ? a.z : b.z, first ? a.w : b.w);
}

template <typename T, int kGroup>
__global__ void __launch_bounds__(kRopeThreads, kRopeResident)
    norm_rope_kernel(RopeParams p, int spans, int span) {
  constexpr int kVec = 16 / sizeof(T), kHeads = 32 / kGroup;
  const int lane = threadIdx.x & 31, j = lane % kGroup;
  const int all = p.heads[0] + p.heads[1], half = p.head_dim / 2;
  const int64_t item = (int64_t)blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
  const int64_t n = item / spans;
  if (n >= p.tokens) return;
  const int first = (int)(item % spans) * span * kHeads + lane / kGroup;
  const int last = min(all, ((int)(item % spans) + 1) * span * kHeads);
  const bool in_head = j * kVec < half;
  const T *in[2] = {static_cast<const T *>(p.in[0]) + n * p.token_stride[0] + j * kVec,
                    static_cast<const T *>(p.in[1]) + n * p.token_stride[1] + j * kVec};

  uint4 lo, hi;
  auto fetch = [&](int h) {
    lo = hi = make_uint4(0, 0, 0, 0);
    if (h < last && in_head) {
      const T *x = h < p.heads[0] ? in[0] + h * p.head_stride[0]
                                  : in[1] + (h - p.heads[0]) * p.head_stride[1];
      lo = __ldcs(reinterpret_cast<const uint4 *>(x));
      hi = __ldcs(reinterpret_cast<const uint4 *>(x + half));
    }
  };
  fetch(first);
  uint4 w_lo[2], w_hi[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const T *w = static_cast<const T *>(p.weight[k]) + j * kVec;
    if (p.weight[k] != nullptr && in_head) {
      w_lo[k] = __ldg(reinterpret_cast<const uint4 *>(w));
      w_hi[k] = __ldg(reinterpret_cast<const uint4 *>(w + half));
    }
  }
  // Angles: kMine a lane, handed round so that every group has its head's. (All of them
  // in every group cost 10 us of 135 at 32,768 tokens of 40 heads.)
  constexpr int kMine = kVec >= kHeads ? kVec / kHeads : 1;
  float2 cosine[kVec / 2], sine[kVec / 2];
  {
    const double position = position_of(p, n);
    float c[kMine], s[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int at = lane * kMine + i;
      c[i] = s[i] = 0.f;
      if (at < half) turn(position, __ldg(p.inv_freq + at), c[i], s[i]);
    }
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {
      const int from = j * (kVec / kMine) + i / kMine, next = j * (kVec / kMine) + (i + 1) / kMine;
      cosine[i / 2] = make_float2(__shfl_sync(kFullMask, c[i % kMine], from),
                                  __shfl_sync(kFullMask, c[(i + 1) % kMine], next));
      sine[i / 2] = make_float2(__shfl_sync(kFullMask, s[i % kMine], from),
                                __shfl_sync(kFullMask, s[(i + 1) % kMine], next));
    }
  }
  // every lane of the warp takes every step: the norms are sums over its group
  for (int h0 = first; h0 - lane / kGroup < last; h0 += kHeads) {
    float2 a[kVec / 2], b[kVec / 2];
    unpack<T, kVec / 2>(lo, a);
    unpack<T, kVec / 2>(hi, b);
    if (h0 - lane / kGroup + kHeads < last) fetch(h0 + kHeads);
    const int h = h0;
    const bool which = h >= p.heads[0];
    float2 squares = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
      squares = pack_fma(a[i], a[i], squares);
      squares = pack_fma(b[i], b[i], squares);
    }
    float sum = squares.x + squares.y;
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
    if (h >= last || !in_head) continue;
    if (p.weight[which] != nullptr) {
      const float scale = rsqrtf(sum / (float)p.head_dim + p.eps);
      const float2 scale2 = make_float2(scale, scale);
      float2 wa[kVec / 2], wb[kVec / 2];
      unpack<T, kVec / 2>(choose(which, w_lo[1], w_lo[0]), wa);
      unpack<T, kVec / 2>(choose(which, w_hi[1], w_hi[0]), wb);
#pragma unroll
      for (int i = 0; i < kVec / 2; ++i) {
        a[i] = pack_mul(a[i], pack_mul(wa[i], scale2));
        b[i] = pack_mul(b[i], pack_mul(wb[i], scale2));
      }
    }
    float2 out_lo[kVec / 2], out_hi[kVec / 2];
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
      const float2 bs = pack_mul(b[i], sine[i]);
      out_lo[i] = pack_fma(a[i], cosine[i], make_float2(-bs.x, -bs.y));
      out_hi[i] = pack_fma(b[i], cosine[i], pack_mul(a[i], sine[i]));
    }
    T *out = static_cast<T *>(p.out[which]) +
             (n * p.heads[which] + (which ? h - p.heads[0] : h)) * p.head_dim + j * kVec;
    *reinterpret_cast<uint4 *>(out) = pack<T, kVec / 2>(out_lo);
    *reinterpret_cast<uint4 *>(out + half) = pack<T, kVec / 2>(out_hi);
  }
}

template <typename T, int kGroup> int launch_vector(const RopeParams &p, cudaStream_t s) {
  // One token's heads are split over `spans` warps so that (rounds of blocks) x (head
  // sets of a warp and its angles, as much as about two) is least: few tokens spread out,
  // many compute their angles once, and the last round is not a nearly empty one.
  const int sets = (int)ceil_div(p.heads[0] + p.heads[1], 32 / kGroup);
  const int64_t places = (int64_t)kRopeResident * sm_count();
  int span = sets, spans = 1;
  int64_t least = 0;
  // a warp for every set where one round holds them
  const bool one_round = p.tokens * sets <= places * kRopeWarps;
  const int from = one_round ? sets : 1, to = one_round ? sets : sets < 64 ? sets : 64;
  for (int n = from; n <= to; ++n) {
    const int each = (int)ceil_div(sets, n), warps = (int)ceil_div(sets, each);
    const int64_t rounds = ceil_div(ceil_div(p.tokens * warps, kRopeWarps), places);
    if (n == from || rounds * (each + 2) < least) {
      least = rounds * (each + 2);
      span = each;
      spans = warps;
    }
  }
  const int64_t blocks = ceil_div(p.tokens * spans, kRopeWarps);
  if (blocks > 0x7fffffff)
    return set_error(HS_ERR_UNSUPPORTED, "norm_rope: too many tokens");
  norm_rope_kernel<T, kGroup><<<(unsigned)blocks, kRopeThreads, 0, s>>>(p, spans, span);
  return check_launch("norm_rope_kernel");
}

template <typename T> int launch(const RopeParams &p, cudaStream_t s) {
  // 16-byte vectors: half a head is a whole number of them, and every address
  // is a multiple of 16 bytes
  constexpr int kVec = 16 / sizeof(T);
  const int half = p.head_dim / 2;
  bool vector = half % kVec == 0;
  for (int k = 0; k < 2; ++k)
    vector = vector && p.token_stride[k] % kVec == 0 && p.head_stride[k] % kVec == 0 &&
             ((reinterpret_cast<uintptr_t>(p.in[k]) | reinterpret_cast<uintptr_t>(p.out[k]) |
               reinterpret_cast<uintptr_t>(p.weight[k])) & 15) == 0;
  if (vector) {
    const int lanes = half / kVec;
    if (lanes <= 4) return launch_vector<T, 4>(p, s);
    if (lanes <= 8) return launch_vector<T, 8>(p, s);
    if constexpr (kVec == 4)  // the largest half holds 32 vectors of fp32
      if (lanes > 16) return launch_vector<T, 32>(p, s);
    return launch_vector<T, 16>(p, s);
  }
  const int64_t blocks = ceil_div(p.tokens * (p.heads[0] + p.heads[1]), kRopeWarps);
  if (blocks > 0x7fffffff)
    return set_error(HS_ERR_UNSUPPORTED, "norm_rope: too many tokens");
  norm_rope_any_kernel<T><<<(unsigned)blocks, kRopeThreads, 0, s>>>(p);
  return check_launch("norm_rope_any_kernel");
}

}  // namespace
}  // namespace hs

extern "C" int hs_qk_norm_rope(int64_t tokens, const void *query, int64_t query_token_stride,
                               int64_t query_head_stride, int q_heads, const void *key,
                               int64_t key_token_stride, int64_t key_head_stride, int kv_heads,
                               int head_dim, int dtype, const void *positions,
                               int positions_dtype, const double *inv_freq,
                               const void *query_weight, const void *key_weight, float eps,
                               void *query_out, void *key_out, hs_stream stream) {
  using namespace hs;
  if (tokens < 0 || q_heads < 1 || kv_heads < 1 || head_dim < 2 || head_dim % 2)
    return set_error(HS_ERR_INVALID_ARGUMENT, "norm_rope: invalid sizes");
  if (head_dim > kRopeMaxDim)
    return set_error(HS_ERR_UNSUPPORTED, "norm_rope: head_dim %d > %d is not supported", head_dim,
                     kRopeMaxDim);
  if (positions_dtype != HS_INT32 && positions_dtype != HS_INT64)
    return set_error(HS_ERR_INVALID_ARGUMENT, "norm_rope: positions must be int32 or int64");
  if (!(eps >= 0.f))
    return set_error(HS_ERR_INVALID_ARGUMENT, "norm_rope: eps must not be negative");
  if (tokens == 0) return HS_OK;
  if (!query || !key || !positions || !inv_freq || !query_out || !key_out)
    return set_error(HS_ERR_INVALID_ARGUMENT, "norm_rope: null pointer");
  const RopeParams p{tokens, {query, key}, {query_token_stride, key_token_stride},
                     {query_head_stride, key_head_stride}, {q_heads, kv_heads},
                     {query_weight, key_weight}, {query_out, key_out}, head_dim, positions,
                     positions_dtype == HS_INT64, inv_freq, eps};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case HS_FLOAT32: return launch<float>(p, s);
    case HS_FLOAT16: return launch<__half>(p, s);
    case HS_BFLOAT16: return launch<__nv_bfloat16>(p, s);
  }
  return set_error(HS_ERR_INVALID_ARGUMENT, "norm_rope: invalid dtype %d", dtype);
}
