// (9) Append to an 8-bit cache, and (10) reading its rows back.
//
// append: one block serves a chunk's K or V of up to 16 KV heads. A head's row is spread
// over kLanes lanes, 8 elements a lane, so that a warp has 32 / kLanes rows of a head at
// once and kBatch such groups of rows in flight: the reads are what bounds it, as long as
// enough of them are on their way. The largest elements meet in shuffles, the exponent
// follows from their bits, the codes leave as 8 bytes a lane. The scales' bytes of a row
// meet in shared memory and are written together with the padding: a byte at a time they
// would be separate transfers over the host link. Bounds and mean come from the values
// held, so that they do not depend on how the rows were split over calls; the page's
// earlier rows are read back for the mean. Where a chunk may have many rows, several
// warps (slices) share a head.
#include "quantized.cuh"

namespace hs {
namespace {

constexpr int kHeadGroup = 16;                  // heads of a block
constexpr int kAppendWarps = 16;                // of a block at most
constexpr int kTailRows = 64;                   // rows whose scales are kept in shared memory
constexpr int kBatch = 4;                       // rows of a lane in flight

struct QuantAppendParams {
  int batch;
  int64_t tokens;
  const void *k, *v;
  int64_t kv_batch_stride;
  const int32_t *within, *count;
  const int64_t *pool_block, *host_block;
  unsigned char *pool, *host;
  int64_t pool_blocks, host_blocks;
  const uint64_t *minimum_ptrs, *maximum_ptrs, *summary_ptrs;
  int kv_heads, head_dim, page_size;
  int64_t record;
  int32_t *status;
};

// This lane's 8 elements of a row as they are in memory
template <typename T> struct Raw {
  uint4 words[sizeof(T) / 2];
  template <bool kWide> __device__ __forceinline__ void load(const T *from, int n) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) words[i] = make_uint4(0, 0, 0, 0);
    if constexpr (kWide) {
      if (n > 0)
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
          words[i] = __ldg(reinterpret_cast<const uint4 *>(from) + i);
    } else {
      T *x = reinterpret_cast<T *>(words);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) x[i] = from[i];
    }
  }
  __device__ __forceinline__ float at(int i) const {
    return to_f32(reinterpret_cast<const T *>(words)[i]);
  }
};
template <bool kWide>
__device__ __forceinline__ void store8(unsigned char *to, int n, uint2 codes) {
  if constexpr (kWide) {
    if (n > 0) *reinterpret_cast<uint2 *>(to) = codes;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) to[i] = (unsigned char)((i < 4 ? codes.x : codes.y) >> (i % 4 * 8));
  }
}
template <bool kWide>
__device__ __forceinline__ uint2 load_codes(const unsigned char *from, int n) {
  uint2 codes = make_uint2(0, 0);
  if constexpr (kWide) {
    if (n > 0) codes = *reinterpret_cast<const uint2 *>(from);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) (i < 4 ? codes.x : codes.y) |= (uint32_t)from[i] << (i % 4 * 8);
  }
  return codes;
}
__device__ __forceinline__ void decode8(uint2 codes, float scale, float (&x)[8]) {
  const float4 lo = decode4_f32(codes.x), hi = decode4_f32(codes.y);
  x[0] = lo.x * scale;
  x[1] = lo.y * scale;
  x[2] = lo.z * scale;
  x[3] = lo.w * scale;
  x[4] = hi.x * scale;
  x[5] = hi.y * scale;
  x[6] = hi.z * scale;
  x[7] = hi.w * scale;
}

// kWide: head_dim is a multiple of 8 and every address of its vector's size
template <typename T, bool kWide, int kLanes>
__global__ void __launch_bounds__(32 * kAppendWarps)
    append_quantized_kernel(QuantAppendParams p, int slices) {
  __shared__ unsigned char scales[kTailRows][kHeadGroup];
  __shared__ float columns[kAppendWarps][8 * kLanes];
  constexpr int kTogether = 32 / kLanes;  // rows of a warp at once
  const int b = blockIdx.y, plane = blockIdx.x & 1, h0 = (blockIdx.x >> 1) * kHeadGroup;
  const int cnt = p.count[b], w = p.within[b];
  const int64_t blk = p.pool_block[b], hb = p.host_block != nullptr ? p.host_block[b] : -1;
  const bool metadata = plane == 0 && p.minimum_ptrs != nullptr;
  uint64_t entries[3] = {0, 0, 0};  // of the page's bounds and mean
  if (metadata) {
    entries[0] = p.minimum_ptrs[b];
    entries[1] = p.maximum_ptrs[b];
    entries[2] = p.summary_ptrs[b];
  }
  if (cnt <= 0) return;
  // pool_block < 0: a host-only chunk (a page with no pool block), which needs a host block
  const bool host_ok = hb >= 0 && p.host != nullptr && hb < p.host_blocks;
  if (w < 0 || cnt > p.page_size - w || cnt > p.tokens || blk >= p.pool_blocks || (hb >= 0 && !host_ok) ||
      (blk < 0 && !host_ok)) {
    if (threadIdx.x == 0) flag(p.status, HS_DEV_ROW_OUT_OF_RANGE);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = p.head_dim;
  const int heads = min(kHeadGroup, p.kv_heads - h0);
  const int head = warp / slices, h = h0 + head, slice = warp - head * slices;
  const bool here = head < heads;
  const int d0 = lane % kLanes * 8, n = here ? min(8, D - d0) : 0;  // this lane's elements
  const int step = slices * kTogether, first = slice * kTogether + lane / kLanes;
  const int64_t E = (int64_t)p.kv_heads * D, at = (int64_t)h * D + d0;
  unsigned char *pool = blk >= 0 ? p.pool + (blk * 2 + plane) * p.page_size * p.record : nullptr;
  unsigned char *host = hb >= 0 ? p.host + (hb * 2 + plane) * p.page_size * p.record : nullptr;
  const T *from = static_cast<const T *>(plane ? p.v : p.k) + (int64_t)b * p.kv_batch_stride + at;

  Raw<T> raw[kBatch];
  const auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int r = i0 + u * step + first;
      raw[u].template load<kWide>(from + (int64_t)r * E, r < cnt ? n : 0);
    }
  };
  load(0);
  // the bounds so far, by the lanes that will write them
  const bool writes = metadata && here && slice == 0 && lane < kLanes && n > 0;
  __nv_bfloat16 *minimum = reinterpret_cast<__nv_bfloat16 *>(entries[0]) + at;
  __nv_bfloat16 *maximum = reinterpret_cast<__nv_bfloat16 *>(entries[1]) + at;
  float low[8], high[8], sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    low[i] = writes && i < n ? __bfloat162float(minimum[i]) : INFINITY;
    high[i] = writes && i < n ? __bfloat162float(maximum[i]) : -INFINITY;
    sum[i] = 0.f;
  }
  if (metadata && here) {  // rows 0 .. w-1 of the page, for the mean
    const unsigned char *page = pool != nullptr ? pool : host;
    for (int r0 = first; r0 < w; r0 += kBatch * step) {
      uint2 codes[kBatch];
      unsigned scale[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const unsigned char *record = page + (int64_t)(r0 + u * step) * p.record;
        const bool is = r0 + u * step < w;
        codes[u] = load_codes<kWide>(record + at, is ? n : 0);
        scale[u] = is ? record[E + h] : 0;
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        float x[8];
        decode8(codes[u], scale_of(scale[u]), x);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += x[i];
      }
    }
  }
  const int tail = (int)(p.record - E);  // bytes of a record behind its codes
  const bool last_group = h0 + heads == p.kv_heads;
  const int own = last_group ? tail - h0 : heads;  // those that this block writes
  for (int r0 = 0; r0 < cnt; r0 += kTailRows) {
    const int rows = min(kTailRows, cnt - r0);
    for (int i0 = 0; i0 < rows; i0 += kBatch * step) {
      if (r0 + i0 > 0) load(r0 + i0);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int r = i0 + u * step + first;
        if (i0 + u * step >= rows) break;  // the same for the whole block
        float x[8], largest = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = raw[u].at(i);
#pragma unroll
        for (int i = 0; i < 8; i += 2) largest = max3_nan(largest, fabsf(x[i]), fabsf(x[i + 1]));
#pragma unroll
        for (int o = kLanes >> 1; o > 0; o >>= 1)
          largest = max_nan(largest, __shfl_xor_sync(kFullMask, largest, o));
        if (!__all_sync(kFullMask, largest < INFINITY)) {  // the largest of the finite ones
          largest = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool finite = fabsf(x[i]) < INFINITY;
            largest = fmaxf(largest, finite ? fabsf(x[i]) : 0.f);
            x[i] = finite ? x[i] : __int_as_float(0x7fffffff);
          }
#pragma unroll
          for (int o = kLanes >> 1; o > 0; o >>= 1)
            largest = fmaxf(largest, __shfl_xor_sync(kFullMask, largest, o));
        }
        const int e = exponent_of(largest);
        const float inverse = power_of_two(-e);
        const uint2 codes =
            make_uint2(encode4(x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse),
                       encode4(x[4] * inverse, x[5] * inverse, x[6] * inverse, x[7] * inverse));
        if (r >= rows || !here) continue;
        const int64_t to = (int64_t)(w + r0 + r) * p.record + at;
        if (pool != nullptr) store8<kWide>(pool + to, n, codes);
        if (host != nullptr) store8<kWide>(host + to, n, codes);
        if (lane % kLanes == 0) scales[r][head] = (unsigned char)(e + 127);
        if (metadata) {
          decode8(codes, power_of_two(e), x);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            low[i] = min_nan(low[i], x[i]);
            high[i] = max_nan(high[i], x[i]);
            sum[i] += x[i];
          }
        }
      }
    }
    __syncthreads();
    // the scales and, by the last group, the padding
    for (int r = warp; r < rows; r += blockDim.x >> 5)
      for (int j = lane; j < own; j += 32) {
        const unsigned char byte = j < heads ? scales[r][j] : 0;
        const int64_t to = (int64_t)(w + r0 + r) * p.record + E + h0 + j;
        if (pool != nullptr) pool[to] = byte;
        if (host != nullptr) host[to] = byte;
      }
    if (r0 + kTailRows < cnt) __syncthreads();
  }
  if (!metadata) return;
  // ---- metadata: the lanes that share columns meet in shuffles, the slices in shared memory
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      low[i] = min_nan(low[i], __shfl_xor_sync(kFullMask, low[i], o));
      high[i] = max_nan(high[i], __shfl_xor_sync(kFullMask, high[i], o));
      sum[i] += __shfl_xor_sync(kFullMask, sum[i], o);
    }
  }
  const auto join = [&](float(&x)[8], auto op) {
    if (slices == 1) return;
    if (lane < kLanes)
#pragma unroll
      for (int i = 0; i < 8; ++i) columns[warp][d0 + i] = x[i];
    __syncthreads();
    if (slice == 0)
      for (int s = 1; s < slices; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = op(x[i], columns[warp + s][d0 + i]);
    __syncthreads();
  };
  join(low, [](float a, float c) { return min_nan(a, c); });
  join(high, [](float a, float c) { return max_nan(a, c); });
  join(sum, [](float a, float c) { return a + c; });
  if (!writes) return;
  float *summary = reinterpret_cast<float *>(entries[2]) + at;
  const float rows = (float)(w + cnt);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= n) break;
    // a value held has 4 significant bits: exact in bf16
    minimum[i] = __float2bfloat16_rn(low[i]);
    maximum[i] = __float2bfloat16_rn(high[i]);
    summary[i] = sum[i] / rows;
  }
}

template <typename T, bool kWide>
int launch_append(const QuantAppendParams &p, int64_t tokens, cudaStream_t s) {
  const int heads = p.kv_heads < kHeadGroup ? p.kv_heads : kHeadGroup;
  int lanes = 4;  // of a head's row
  while (lanes * 8 < p.head_dim) lanes <<= 1;
  // Slices while a lane still has a batch of rows (2,048 pages of 16 rows, 8 heads of 128:
  // one slice) and the block has warps left.
  int slices = 1;
  while (2 * slices * heads <= kAppendWarps && slices * (32 / lanes) * kBatch * 2 < tokens)
    slices *= 2;
  const dim3 grid((unsigned)(2 * ceil_div(p.kv_heads, kHeadGroup)), (unsigned)p.batch);
  const int threads = 32 * heads * slices;
  switch (lanes) {
    case 4: append_quantized_kernel<T, kWide, 4><<<grid, threads, 0, s>>>(p, slices); break;
    case 8: append_quantized_kernel<T, kWide, 8><<<grid, threads, 0, s>>>(p, slices); break;
    case 16: append_quantized_kernel<T, kWide, 16><<<grid, threads, 0, s>>>(p, slices); break;
    default: append_quantized_kernel<T, kWide, 32><<<grid, threads, 0, s>>>(p, slices); break;
  }
  return check_launch("append_quantized_kernel");
}
template <typename T>
int launch_append(const QuantAppendParams &p, int64_t tokens, cudaStream_t s) {
  const uintptr_t in = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                       (uintptr_t)(p.kv_batch_stride * (int64_t)sizeof(T));
  const uintptr_t held = reinterpret_cast<uintptr_t>(p.pool) | reinterpret_cast<uintptr_t>(p.host);
  const bool wide = p.head_dim % 8 == 0 && in % 16 == 0 && held % 8 == 0;
  return wide ? launch_append<T, true>(p, tokens, s) : launch_append<T, false>(p, tokens, s);
}

// ---- (10) ---------------------------------------------------------------------------------
constexpr int kReadThreads = 256;
constexpr int kReadRows = 16;   // rows of a block
constexpr int kReadAhead = 4;   // loads in flight

struct ReadParams {
  const unsigned char *pool;
  int64_t pool_blocks;
  const int64_t *rows;
  int64_t count;
  void *out;
  int kv_heads, head_dim, page_size, page_shift;
  int64_t record;
  int32_t *status;
};

template <typename T> struct alignas(8 * sizeof(T) < 16 ? 8 * sizeof(T) : 16) Eight { T x[8]; };

// kN codes a thread and step: 8, or 1 where head_dim or an address does not allow it
template <typename T, int kN>
__global__ void __launch_bounds__(kReadThreads) read_quantized_kernel(ReadParams p) {
  __shared__ int64_t records[kReadRows];  // index of the K record, or -1
  const int64_t row0 = (int64_t)blockIdx.x * kReadRows;
  const int rows = (int)min((int64_t)kReadRows, p.count - row0);
  if (threadIdx.x < rows)
    records[threadIdx.x] = record_index(p.rows[row0 + threadIdx.x], p.page_size, p.page_shift,
                                        p.pool_blocks, p.status);
  __syncthreads();
  const int64_t E = (int64_t)p.kv_heads * p.head_dim;
  const int units = (int)(E / kN), per_head = p.head_dim / kN;
  T *out = static_cast<T *>(p.out);
  for (int plane = 0; plane < 2; ++plane) {
    const int all = rows * units;
    for (int i0 = threadIdx.x; i0 < all; i0 += kReadThreads * kReadAhead) {
      uint2 codes[kReadAhead];
      unsigned scale[kReadAhead];
#pragma unroll
      for (int u = 0; u < kReadAhead; ++u) {
        const int i = i0 + u * kReadThreads, r = i / units, c = i - r * units;
        codes[u] = make_uint2(0, 0);
        scale[u] = 127;
        if (i < all && records[r] >= 0) {
          const unsigned char *record =
              p.pool + (records[r] + (int64_t)plane * p.page_size) * p.record;
          if constexpr (kN == 8) codes[u] = __ldg(reinterpret_cast<const uint2 *>(record) + c);
          else codes[u].x = record[c];
          scale[u] = record[E + c / per_head];
        }
      }
#pragma unroll
      for (int u = 0; u < kReadAhead; ++u) {
        const int i = i0 + u * kReadThreads;
        if (i >= all) break;
        float x[8];
        decode8(codes[u], scale_of(scale[u]), x);
        T *to = out + ((int64_t)plane * p.count + row0) * E + (int64_t)i * kN;
        if constexpr (kN == 8) {
          Eight<T> y;
#pragma unroll
          for (int j = 0; j < 8; ++j) y.x[j] = from_f32<T>(x[j]);
          *reinterpret_cast<Eight<T> *>(to) = y;
        } else {
          *to = from_f32<T>(x[0]);
        }
      }
    }
  }
}

template <typename T> int launch_read(const ReadParams &p, cudaStream_t s) {
  const unsigned grid = (unsigned)ceil_div(p.count, kReadRows);
  const bool wide = p.head_dim % 8 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  if (wide) read_quantized_kernel<T, 8><<<grid, kReadThreads, 0, s>>>(p);
  else read_quantized_kernel<T, 1><<<grid, kReadThreads, 0, s>>>(p);
  return check_launch("read_quantized_kernel");
}

}  // namespace
}  // namespace hs

extern "C" int64_t hs_quantized_row_bytes(int kv_heads, int head_dim) {
  if (kv_heads < 1 || head_dim < 1) return 0;
  return hs::record_bytes(kv_heads, head_dim);
}

extern "C" int hs_append_quantized(int batch, int64_t tokens, const void *k, const void *v,
                                   int64_t kv_batch_stride, int kv_dtype, const int32_t *within,
                                   const int32_t *count, const int64_t *pool_block, void *pool,
                                   int64_t pool_blocks, const int64_t *host_block,
                                   void *host_alias, int64_t host_blocks,
                                   const uint64_t *minimum_ptrs, const uint64_t *maximum_ptrs,
                                   const uint64_t *summary_ptrs, int kv_heads, int head_dim,
                                   int page_size, int32_t *device_status, hs_stream stream) {
  using namespace hs;
  if (batch < 0 || tokens < 0 || kv_heads < 1 || head_dim < 1 || page_size < 1 ||
      pool_blocks < 0 || host_blocks < 0 || kv_batch_stride < 0)
    return set_error(HS_ERR_INVALID_ARGUMENT, "append: invalid sizes");
  if (kv_dtype != HS_FLOAT32 && kv_dtype != HS_FLOAT16 && kv_dtype != HS_BFLOAT16)
    return set_error(HS_ERR_INVALID_ARGUMENT, "append: invalid KV dtype %d", kv_dtype);
  if (head_dim > kQuantMaxDim)
    return set_error(HS_ERR_UNSUPPORTED, "append: head_dim %d > %d is not supported", head_dim,
                     kQuantMaxDim);
  if (batch == 0 || tokens == 0) return HS_OK;
  if (!k || !v || !within || !count || !pool_block || !pool ||
      !minimum_ptrs != !maximum_ptrs || !minimum_ptrs != !summary_ptrs)
    return set_error(HS_ERR_INVALID_ARGUMENT, "append: null pointer");
  if (batch > 65535) return set_error(HS_ERR_UNSUPPORTED, "append: batch %d > 65535", batch);
  QuantAppendParams p{batch, tokens, k, v, kv_batch_stride, within, count, pool_block, host_block,
                      static_cast<unsigned char *>(pool),
                      static_cast<unsigned char *>(host_alias), pool_blocks, host_blocks,
                      minimum_ptrs, maximum_ptrs, summary_ptrs, kv_heads, head_dim, page_size,
                      record_bytes(kv_heads, head_dim), device_status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (kv_dtype) {
    case HS_FLOAT32: return launch_append<float>(p, tokens, s);
    case HS_FLOAT16: return launch_append<__half>(p, tokens, s);
    default: return launch_append<__nv_bfloat16>(p, tokens, s);
  }
}

extern "C" int hs_read_quantized(const void *pool, int64_t pool_blocks, const int64_t *rows,
                                 int64_t count, void *out, int dtype, int kv_heads, int head_dim,
                                 int page_size, int32_t *device_status, hs_stream stream) {
  using namespace hs;
  if (kv_heads < 1 || head_dim < 1 || page_size < 1 || pool_blocks < 0 || count < 0)
    return set_error(HS_ERR_INVALID_ARGUMENT, "read_quantized: invalid sizes");
  if (dtype != HS_FLOAT32 && dtype != HS_FLOAT16 && dtype != HS_BFLOAT16)
    return set_error(HS_ERR_INVALID_ARGUMENT, "read_quantized: invalid dtype %d", dtype);
  if (head_dim > kQuantMaxDim)
    return set_error(HS_ERR_UNSUPPORTED, "read_quantized: head_dim %d > %d is not supported",
                     head_dim, kQuantMaxDim);
  if (count == 0) return HS_OK;
  if (!pool || !rows || !out)
    return set_error(HS_ERR_INVALID_ARGUMENT, "read_quantized: null pointer");
  if ((reinterpret_cast<uintptr_t>(pool) & 15) != 0)
    return set_error(HS_ERR_INVALID_ARGUMENT, "read_quantized: the pool must be 16-byte aligned");
  if (count > (int64_t)0x7fffffff * kReadRows || (int64_t)kv_heads * head_dim > (1 << 26))
    return set_error(HS_ERR_UNSUPPORTED, "read_quantized: rows or heads too many");
  ReadParams p{static_cast<const unsigned char *>(pool), pool_blocks, rows, count, out, kv_heads,
               head_dim, page_size, page_shift_of(page_size), record_bytes(kv_heads, head_dim),
               device_status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case HS_FLOAT32: return launch_read<float>(p, s);
    case HS_FLOAT16: return launch_read<__half>(p, s);
    default: return launch_read<__nv_bfloat16>(p, s);
  }
}
