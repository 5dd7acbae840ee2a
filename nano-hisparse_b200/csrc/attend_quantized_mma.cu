// Decode attention over an 8-bit cache, 16-bit queries, head_dim a multiple of 16, heads
// that share their rows.
//
// A warp serves one KV head and up to 8 * kTiles of its query heads over tiles of 16
// rows, alone: it copies its own tiles (cp.async, 16 bytes a lane, into a ring of its
// own) and keeps its own maximum, sum and output, so that nothing in the loop waits for
// another warp. The heads of a block read neighbouring parts of the same rows. With
// keys as the M side of m16n8k16 and the query heads as N,
//   S^T = K Q^T     the codes of a lane's ldmatrix word are two fp16 pairs (every e4m3
//                   number is one of fp16); which element of head_dim stands where in
//                   the sum does not matter as long as Q is laid out alike. Q is fp16,
//                   scaled by a power of two for each query, which keeps bf16 exact.
//   O^T += V^T P^T  V through ldmatrix.trans, whose 16-bit unit is two neighbouring
//                   elements of a row: a byte permutation makes pairs of rows of each.
//                   P is rounded to fp16, times 2^7 at the current maximum, which is
//                   raised only when a weight would pass it by more than 2^8. Half a step
//                   of a weight (2^-11) is an eighth of a bf16 result's own rounding; for
//                   fp16 results, which round by as much, what was lost is a second P.
#include <type_traits>

#include "attend_quantized.cuh"

namespace hs {
namespace {

constexpr int kMmaWarps = 8, kMmaThreads = 32 * kMmaWarps;
constexpr int kMmaRows = 16;     // rows of a tile
constexpr float kRaise = 8.f;    // the maximum is raised past this
constexpr float kWeightLift = 7.f;

template <int kDim, int kTiles> struct MmaShape {
  static constexpr int pitch = kDim + 16;  // of a row: an odd number of 16-byte chunks
  static constexpr int plane = kMmaRows * pitch;
  static constexpr int stage = 2 * plane + 2 * kMmaRows * 4;  // K, V, the words with their scales
  static constexpr int stages = kDim == 64 ? 4 : 3;
  static constexpr int resident = kDim <= 128 && kTiles == 1 ? 2 : 1;
  static constexpr int queries = 8 * kTiles;
  static constexpr int ring = stages * stage;
  // the warps' results at the end, in the place of the rings
  static constexpr int result = queries * (kDim + 4) * 4;
  static constexpr size_t bytes = (size_t)kMmaWarps * (ring > result ? ring : result);
  static_assert(resident * (bytes + 1024) <= 228 * 1024, "the blocks fit an SM");
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // an 8 x 8 matrix of 16 bits
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// bytes: 0 leaves zeros and reads nothing
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}

template <typename T, int kDim, int kTiles>
__global__ void __launch_bounds__(kMmaThreads, MmaShape<kDim, kTiles>::resident)
    quant_mma_kernel(QuantAttendParams p, int heads_of_block, int head_places) {
  using Shape = MmaShape<kDim, kTiles>;
  constexpr int kParts = std::is_same<T, __half>::value ? 2 : 1;  // of P
  constexpr int kChunks = kDim / 16, kQueries = Shape::queries, kStages = Shape::stages;
  extern __shared__ __align__(128) unsigned char smem[];
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = p.head_dim;
  const int split = blockIdx.x, b = blockIdx.z;
  const int chunks = (p.groups + kQueries - 1) / kQueries;  // of a KV head's query heads
  const int group = blockIdx.y / chunks, chunk = blockIdx.y - group * chunks;
  const int slices = kMmaWarps / head_places;  // warps that share a head's rows
  const int place = warp % head_places, slice = warp / head_places;
  const int kh = group * heads_of_block + place;
  const bool here = place < heads_of_block && kh < p.kv_heads;
  const int h0 = kh * p.groups + chunk * kQueries;
  const int hn = here ? min(kQueries, p.groups - chunk * kQueries) : 0;  // query heads

  // this warp's tiles: first, first + slices, ... < last
  const int valid = (int)quant_rows(p, b), tiles = (valid + kMmaRows - 1) / kMmaRows;
  const int first = (int)((int64_t)tiles * split / p.splits) + slice;
  const int last = here ? (int)((int64_t)tiles * (split + 1) / p.splits) : 0;

  const unsigned char *pool = p.pool + (int64_t)kh * D;
  const int64_t E = (int64_t)p.kv_heads * D, v_plane = (int64_t)p.page_size * p.record;
  const int64_t scales = E - (int64_t)kh * D + (kh & ~3);  // of the scales' word, from `pool`
  const int64_t *rows = p.rows + b * p.rows_batch_stride;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * Shape::ring;
  const int c16 = lane % kChunks * 16;
  // a lane has the row number of one row of a tile, read one tile before its copies
  const auto look = [&](int tile) -> int64_t {
    const int at = tile * kMmaRows + (lane & 15);
    return tile < last && at < valid ? __ldg(rows + at) : -1;
  };
  int64_t next = look(first);
  int issue = first, to = 0;  // the next tile to copy and its stage
  const auto copy_tile = [&] {
    if (issue < last) {
      const int64_t index =
          record_index(next, p.page_size, p.page_shift, p.pool_blocks, p.status);
      const int64_t offset = index < 0 ? -1 : index * p.record;
      next = look(issue + slices);
      const uint32_t stage = ring + to * Shape::stage;
      constexpr int together = 32 / kChunks;
#pragma unroll
      for (int i = 0; i < kMmaRows / together; ++i) {
        const int r = i * together + lane / kChunks;
        const int64_t from = __shfl_sync(kFullMask, offset, r);
        const int bytes = from >= 0 && c16 < D ? 16 : 0;
        const unsigned char *src = bytes ? pool + from + c16 : p.pool;
        const uint32_t dst = stage + r * Shape::pitch + c16;
        copy16(dst, src, bytes);
        copy16(dst + Shape::plane, bytes ? src + v_plane : p.pool, bytes);
      }
      // lanes 0-15 the words with the K scales, 16-31 those of V
      const unsigned char *src = pool + offset + scales + (lane < 16 ? 0 : v_plane);
      copy4(stage + 2 * Shape::plane + lane * 4, offset >= 0 ? src : p.pool, offset >= 0 ? 4 : 0);
      issue += slices;
      if (++to == kStages) to = 0;
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) copy_tile();

  // Q: query head lane / 4, of every 16 elements those at 4 * (lane % 4) on
  uint32_t q[kTiles][kChunks][2];
  float factor[kTiles][2];  // of the scores of the query heads 2 * (lane % 4) + 0, 1
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const int g = n * 8 + lane / 4;
    const T *from = static_cast<const T *>(p.query) + (int64_t)b * p.q_batch_stride +
                    (int64_t)(h0 + g) * D + lane % 4 * 4;
    float largest = 0.f;
    uint2 raw[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      raw[c] = make_uint2(0, 0);
      if (g < hn && c * 16 < D) raw[c] = __ldg(reinterpret_cast<const uint2 *>(from + c * 16));
      const T *x = reinterpret_cast<const T *>(&raw[c]);
#pragma unroll
      for (int i = 0; i < 4; ++i) largest = fmaxf(largest, fabsf(to_f32(x[i])));
    }
    largest = fmaxf(largest, __shfl_xor_sync(kFullMask, largest, 1));
    largest = fmaxf(largest, __shfl_xor_sync(kFullMask, largest, 2));
    // to below 2^14: what is 2^27 times smaller is still a normal number of fp16
    const int e = largest > 0.f ? (__float_as_int(largest) >> 23) - 127 - 13 : 0;
    const float scale = power_of_two(max(-126, min(127, -e)));
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const T *x = reinterpret_cast<const T *>(&raw[c]);
      q[n][c][0] = pack_half(to_f32(x[0]) * scale, to_f32(x[1]) * scale);
      q[n][c][1] = pack_half(to_f32(x[2]) * scale, to_f32(x[3]) * scale);
    }
    const float back = p.scale_log2 / scale;
    factor[n][0] = __shfl_sync(kFullMask, back, lane % 4 * 8);
    factor[n][1] = __shfl_sync(kFullMask, back, lane % 4 * 8 + 4);
  }

  float m[kTiles][2], l[kTiles][2], o[kTiles][kChunks][4];
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[n][j] = -INFINITY;
      l[n][j] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][c][i] = 0.f;
  }
  // ldmatrix: matrix lane / 8 has rows (lane / 8 % 2) * 8 on, chunk lane / 16
  const uint32_t matrix = (lane & 15) * Shape::pitch + lane / 16 * 16;
  int slot = 0;
  for (int tile = first; tile < last; tile += slices) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    copy_tile();
    const uint32_t stage = ring + slot * Shape::stage;
    const unsigned char *bytes = smem + warp * Shape::ring + slot * Shape::stage +
                                 2 * Shape::plane + (kh & 3) + lane / 4 * 4;
    if (++slot == kStages) slot = 0;
    // ---- S^T: rows lane / 4 and lane / 4 + 8, query heads 2 * (lane % 4) + 0, 1
    float s[kTiles][2][4];
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][0][i] = s[n][1][i] = 0.f;
#pragma unroll
    for (int c = 0; c < kChunks; c += 2) {
      uint32_t k[4];
      ldmatrix4(k, stage + matrix + c * 16);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint2 lo = decode4(k[2 * u]), hi = decode4(k[2 * u + 1]);
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
          mma_f16(s[n][u], lo.x, hi.x, lo.y, hi.y, q[n][c + u][0], q[n][c + u][1]);
      }
    }
    // a row that is not seen has zeros in the place of its scale, which is never 0
    const unsigned ek[2] = {bytes[0], bytes[32]}, ev[2] = {bytes[64], bytes[96]};
    const float k_scale[2] = {scale_of(ek[0]), scale_of(ek[1])};
    const float v_exponent[2] = {(float)((int)ev[0] - 127), (float)((int)ev[1] - 127)};
    float t[kTiles][4];  // s + exponent
    bool raise = false;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i >> 1, j = i & 1;
        const float x = (s[n][0][i] + s[n][1][i]) * (k_scale[r] * factor[n][j]);
        s[n][0][i] = ek[r] != 0 ? x : -INFINITY;
        t[n][i] = s[n][0][i] + v_exponent[r];
        raise = raise || t[n][i] > m[n][j] + kRaise;
      }
    if (__any_sync(kFullMask, raise)) {
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = fmaxf(t[n][j], t[n][2 + j]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, x));
          top = fmaxf(top, m[n][j]);
          const float f = m[n][j] == -INFINITY ? 0.f : quant_exp2(m[n][j] - top);
          m[n][j] = top;
          l[n][j] *= f;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            o[n][c][j] *= f;
            o[n][c][2 + j] *= f;
          }
        }
    }
    uint32_t w[kTiles][kParts][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      // nothing seen so far: exp2(-inf) = 0
      const float base[2] = {m[n][0] == -INFINITY ? 0.f : kWeightLift - m[n][0],
                             m[n][1] == -INFINITY ? 0.f : kWeightLift - m[n][1]};
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float2 x = make_float2(quant_exp2(t[n][2 * r] + base[0]),
                                     quant_exp2(t[n][2 * r + 1] + base[1]));
        const uint32_t rounded = pack_half(x.x, x.y);
        w[n][0][r] = transpose8(rounded);
        if constexpr (kParts == 2) {
          const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&rounded));
          w[n][1][r] = transpose8(pack_half(x.x - y.x, x.y - y.y));
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) l[n][j] += quant_exp2(s[n][0][2 * r + j] + (base[j] + kSumLift));
      }
    }
    // ---- O^T: elements 16 c + 2 * (lane / 4) + 0, 1, query heads 2 * (lane % 4) + 0, 1
#pragma unroll
    for (int c = 0; c < kChunks; c += 2) {
      uint32_t v[4];
      ldmatrix4_trans(v, stage + Shape::plane + matrix + c * 16);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint2 lo = decode4(__byte_perm(v[2 * u], 0, 0x3120));
        const uint2 hi = decode4(__byte_perm(v[2 * u + 1], 0, 0x3120));
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int part = 0; part < kParts; ++part)
            mma_f16(o[n][c + u], lo.x, lo.y, hi.x, hi.y, w[n][part][0], w[n][part][1]);
      }
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");

  // ---- results --------------------------------------------------------------------------
  const auto write = [&](int g, int d, float top, float sum, float2 x) {
    const int h = h0 + g;
    if (p.out != nullptr) {
      const float inv = sum > 0.f || sum != sum ? kSumScale / sum : 0.f;
      T *out = static_cast<T *>(p.out) + ((int64_t)b * p.q_heads + h) * D + d;
      out[0] = from_f32<T>(x.x * inv);
      out[1] = from_f32<T>(x.y * inv);
    } else {
      const int64_t part = quant_part(p, p.phase, b, h, split);
      if (d == 0) p.stats[part] = make_float4(top, 0.f, sum, 0.f);
      *reinterpret_cast<float2 *>(p.partials + part * quant_pad(D) + d) = x;
    }
  };
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(kFullMask, l[n][j], x);
      m[n][j] -= kWeightLift;
    }
  if (slices == 1) {
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int g = n * 8 + lane % 4 * 2 + j, d = c * 16 + lane / 4 * 2;
          if (g < hn && d < D)
            write(g, d, m[n][j], l[n][j], make_float2(o[n][c][j], o[n][c][2 + j]));
        }
    return;
  }
  // the slices' results meet in shared memory: a query's maximum and sum, then its elements
  __syncthreads();
  float *mine = reinterpret_cast<float *>(smem + (size_t)warp * Shape::result);
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float *to_query = mine + (n * 8 + lane % 4 * 2 + j) * (kDim + 4);
      if (lane < 4) *reinterpret_cast<float2 *>(to_query) = make_float2(m[n][j], l[n][j]);
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        *reinterpret_cast<float2 *>(to_query + 4 + c * 16 + lane / 4 * 2) =
            make_float2(o[n][c][j], o[n][c][2 + j]);
    }
  __syncthreads();
  if (hn == 0) return;
  // warp (place, slice) takes every slices-th query of its head
  for (int g = slice; g < hn; g += slices) {
    const auto of = [&](int s) {
      return reinterpret_cast<const float *>(smem + (size_t)(s * head_places + place) *
                                                        Shape::result) + g * (kDim + 4);
    };
    float top = -INFINITY, sum = 0.f;
    for (int s = 0; s < slices; ++s) top = fmaxf(top, of(s)[0]);
    for (int s = 0; s < slices; ++s)
      if (of(s)[1] != 0.f) sum = fmaf(of(s)[1], quant_exp2(of(s)[0] - top), sum);
    for (int d = lane * 2; d < D; d += 64) {
      float2 x = make_float2(0.f, 0.f);
      for (int s = 0; s < slices; ++s) {
        if (of(s)[1] == 0.f) continue;  // saw nothing
        const float f = quant_exp2(of(s)[0] - top);
        const float2 y = *reinterpret_cast<const float2 *>(of(s) + 4 + d);
        x.x = fmaf(f, y.x, x.x);
        x.y = fmaf(f, y.y, x.y);
      }
      write(g, d, top, sum, x);
    }
  }
}

template <typename T, int kDim, int kTiles>
int launch(const QuantAttendParams &p, cudaStream_t s) {
  auto kernel = quant_mma_kernel<T, kDim, kTiles>;
  const size_t bytes = MmaShape<kDim, kTiles>::bytes;
  if (int e = reserve_smem(reinterpret_cast<const void *>(kernel), bytes, "attend_quantized"))
    return e;
  const QuantMmaGrid g = quant_mma_grid(p.q_heads, p.kv_heads, p.head_dim);
  const dim3 grid((unsigned)p.splits, (unsigned)(g.groups * g.chunks), (unsigned)p.batch);
  kernel<<<grid, kMmaThreads, bytes, s>>>(p, g.heads, g.places);
  return check_launch("quant_mma_kernel");
}
template <typename T> int launch(const QuantAttendParams &p, cudaStream_t s) {
  const bool two = quant_mma_grid(p.q_heads, p.kv_heads, p.head_dim).queries == 16;
  if (p.head_dim <= 64) return two ? launch<T, 64, 2>(p, s) : launch<T, 64, 1>(p, s);
  if (p.head_dim <= 128) return two ? launch<T, 128, 2>(p, s) : launch<T, 128, 1>(p, s);
  return launch<T, 256, 1>(p, s);
}

}  // namespace

QuantMmaGrid quant_mma_grid(int q_heads, int kv_heads, int head_dim) {
  QuantMmaGrid g;
  const int per = q_heads / kv_heads;
  g.queries = per > 8 && head_dim <= 128 ? 16 : 8;
  g.chunks = (per + g.queries - 1) / g.queries;
  g.groups = (kv_heads + kMmaWarps - 1) / kMmaWarps;
  g.heads = (kv_heads + g.groups - 1) / g.groups;
  g.groups = (kv_heads + g.heads - 1) / g.heads;
  for (g.places = 1; g.places < g.heads; g.places <<= 1) {}
  g.resident = head_dim <= 128 && g.queries == 8 ? 2 : 1;
  g.slices = kMmaWarps / g.places;
  return g;
}

int launch_quant_mma(const QuantAttendParams &p, int dtype, cudaStream_t s) {
  return dtype == HS_FLOAT16 ? launch<__half>(p, s) : launch<__nv_bfloat16>(p, s);
}

}  // namespace hs
