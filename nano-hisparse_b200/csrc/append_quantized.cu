// (9) Append to an 8-bit cache, and (10) reading its rows back.
//
// append: one block serves a chunk's K or V of up to 8 KV heads. A head's row is spread
// over kLanes lanes, 8 elements a lane, so that a warp has 32 / kLanes rows of a head at
// once and kBatch such groups of rows in flight. The largest elements meet in shuffles, the exponent
// follows from their bits, the codes leave as 8 bytes a lane. The scales' bytes of a row
// meet in shared memory and are written together with the padding: a byte at a time they
// would be separate transfers over the host link. Bounds and mean come from the values
// held, so that they do not depend on how the rows were split over calls (the mean but for
// the order of its sum); the page's earlier rows are read back for the mean. Where a chunk
// may have many rows, several warps (slices) share a head.
//
// A prompt (2,048 pages of 16 rows, 8 heads of 128, bf16: 227 MB) takes 61 us, 57 % of a
// copy's rate. Its instructions bound it, about 170 for two rows of a head (issue slots
// busy 70 %, the integer pipe 56 %): unpacking, the largest element, the codes and, for K,
// their values and bounds. With one row in flight it took 142, four rows 112; bounds in
// pairs of bf16 halve their instructions and leave registers for four blocks an SM (three: 70;
// five with half the rows in flight: 63). A decode step (a row of each of 16 requests) takes
// 4.5 us with its launch: row and bounds are read side by side, behind one wait for the page.
#include "quantized.cuh"

namespace hs {
namespace {

constexpr int kHeadGroup = 8;                   // heads of a block
constexpr int kAppendWarps = 8;                 // of a block at most
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

// This lane's 8 elements of a row as they are in memory, the first n
template <typename T> struct Raw {
  uint4 words[sizeof(T) / 2];
  template <bool kWide> __device__ __forceinline__ void load(const T *from, int n) {
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        words[i] = __ldg(reinterpret_cast<const uint4 *>(from) + i);
    } else {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) words[i] = make_uint4(0, 0, 0, 0);
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
__device__ __forceinline__ void decode8(uint2 codes, float scale, float2 (&x)[4]) {
  const float4 lo = decode4_f32(codes.x), hi = decode4_f32(codes.y);
  const float2 s = make_float2(scale, scale);
  x[0] = pack_mul(make_float2(lo.x, lo.y), s);
  x[1] = pack_mul(make_float2(lo.z, lo.w), s);
  x[2] = pack_mul(make_float2(hi.x, hi.y), s);
  x[3] = pack_mul(make_float2(hi.z, hi.w), s);
}

// A lane's part of the bounds and sums
struct Columns {
  __nv_bfloat162 low[4], high[4];
  float2 sum[4];
};

// kWide: head_dim is a multiple of 8 and every address of its vector's size
template <typename T, bool kWide, int kLanes>
__global__ void __launch_bounds__(32 * kAppendWarps, sizeof(T) == 2 ? 4 : 2)
    append_quantized_kernel(QuantAppendParams p, int slices) {
  __shared__ unsigned char scales[kTailRows][kHeadGroup];
  __shared__ Columns columns[kAppendWarps][kLanes];
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
  // Rows r, r + step, ... Nothing is read past the last row, nor by lanes and warps past the
  // row's end and the last head: they read what others read and write nothing, and their
  // row's largest element is the same.
  const int row_size = (int)E, record_size = (int)p.record;
  const T *load_from = kWide && n <= 0 ? from - (here ? d0 : at) : from;
  const auto load = [&](int r) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      raw[u].template load<kWide>(load_from + (int64_t)min(r + u * step, cnt - 1) * row_size, n);
  };
  load(first);
  // the bounds so far, by the lanes that will write them
  const bool writes = metadata && here && slice == 0 && lane < kLanes && n > 0;
  __nv_bfloat16 *minimum = reinterpret_cast<__nv_bfloat16 *>(entries[0]) + at;
  __nv_bfloat16 *maximum = reinterpret_cast<__nv_bfloat16 *>(entries[1]) + at;
  // two columns a word: a value held has 4 significant bits and is exact in bf16
  alignas(16) __nv_bfloat162 low[4], high[4];
  float2 sum[4];
  const bool vectors = kWide && ((entries[0] | entries[1] | entries[2]) & 15) == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    low[i] = __float2bfloat162_rn(INFINITY);
    high[i] = __float2bfloat162_rn(-INFINITY);
  }
  if (writes) {
    if (vectors) {
      *reinterpret_cast<uint4 *>(low) = *reinterpret_cast<const uint4 *>(minimum);
      *reinterpret_cast<uint4 *>(high) = *reinterpret_cast<const uint4 *>(maximum);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) {
          reinterpret_cast<__nv_bfloat16 *>(low)[i] = minimum[i];
          reinterpret_cast<__nv_bfloat16 *>(high)[i] = maximum[i];
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sum[i] = make_float2(0.f, 0.f);
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
        float2 x[4];
        decode8(codes[u], scale_of(scale[u]), x);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = pack_add(sum[i], x[i]);
      }
    }
  }
  const int tail = (int)(p.record - E);  // bytes of a record behind its codes
  const bool last_group = h0 + heads == p.kv_heads;
  const int own = last_group ? tail - h0 : heads;  // those that this block writes
  // where the next row goes
  const int64_t place = (int64_t)w * p.record + at;
  unsigned char *pool_at = pool != nullptr ? pool + place : nullptr;
  unsigned char *host_at = host != nullptr ? host + place : nullptr;
  for (int r0 = 0; r0 < cnt; r0 += kTailRows) {
    const int rows = min(kTailRows, cnt - r0);
    for (int i0 = 0; i0 < rows; i0 += kBatch * step) {
      if (r0 + i0 > 0) load(r0 + i0 + first);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (i0 + u * step >= rows) break;  // the same for the whole block
        const int r = i0 + u * step + first;  // of the tile
        float2 x[4];
        float largest = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = make_float2(raw[u].at(2 * i), raw[u].at(2 * i + 1));
          largest = max3_nan(largest, fabsf(x[i].x), fabsf(x[i].y));
        }
#pragma unroll
        for (int o = kLanes >> 1; o > 0; o >>= 1)
          largest = max_nan(largest, __shfl_xor_sync(kFullMask, largest, o));
        if (!__all_sync(kFullMask, largest < INFINITY)) {  // the largest of the finite ones
          largest = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float nan = __int_as_float(0x7fffffff);
            if (!(fabsf(x[i].x) < INFINITY)) x[i].x = nan;
            if (!(fabsf(x[i].y) < INFINITY)) x[i].y = nan;
            largest = fmaxf(largest, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));  // ignores NaN
          }
#pragma unroll
          for (int o = kLanes >> 1; o > 0; o >>= 1)
            largest = fmaxf(largest, __shfl_xor_sync(kFullMask, largest, o));
        }
        const int e = exponent_of(largest);
        const float2 inverse = make_float2(power_of_two(-e), power_of_two(-e));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = pack_mul(x[i], inverse);
        const uint2 codes = make_uint2(encode4(x[0].x, x[0].y, x[1].x, x[1].y),
                                       encode4(x[2].x, x[2].y, x[3].x, x[3].y));
        if (r >= rows || !here) continue;
        const int64_t to = (int64_t)(r0 + r) * record_size;
        if (pool != nullptr) store8<kWide>(pool_at + to, n, codes);
        if (host != nullptr) store8<kWide>(host_at + to, n, codes);
        if (lane % kLanes == 0) scales[r][head] = (unsigned char)(e + 127);
        if (metadata) {
          decode8(codes, power_of_two(e), x);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 y = __floats2bfloat162_rn(x[i].x, x[i].y);
            low[i] = __hmin2_nan(low[i], y);
            high[i] = __hmax2_nan(high[i], y);
            sum[i] = pack_add(sum[i], x[i]);
          }
        }
      }
    }
    __syncthreads();
    // the scales and, by the last group, the padding
    const int64_t row0 = (int64_t)(w + r0) * p.record + E + h0;
    for (int r = warp; r < rows; r += blockDim.x >> 5)
      for (int j = lane; j < own; j += 32) {
        const unsigned char byte = j < heads ? scales[r][j] : 0;
        if (pool != nullptr) pool[row0 + r * p.record + j] = byte;
        if (host != nullptr) host[row0 + r * p.record + j] = byte;
      }
    if (r0 + kTailRows < cnt) __syncthreads();
  }
  if (!metadata) return;
  // ---- metadata: the lanes that share columns meet in shuffles, the slices in shared memory
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      low[i] = __hmin2_nan(low[i], __shfl_xor_sync(kFullMask, low[i], o));
      high[i] = __hmax2_nan(high[i], __shfl_xor_sync(kFullMask, high[i], o));
      sum[i].x += __shfl_xor_sync(kFullMask, sum[i].x, o);
      sum[i].y += __shfl_xor_sync(kFullMask, sum[i].y, o);
    }
  }
  if (slices > 1) {
    Columns &mine = columns[warp][lane % kLanes];
    if (slice > 0 && lane < kLanes)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mine.low[i] = low[i];
        mine.high[i] = high[i];
        mine.sum[i] = sum[i];
      }
    __syncthreads();
    if (slice == 0)
      for (int s = 1; s < slices; ++s) {
        const Columns &other = columns[warp + s][lane % kLanes];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          low[i] = __hmin2_nan(low[i], other.low[i]);
          high[i] = __hmax2_nan(high[i], other.high[i]);
          sum[i] = pack_add(sum[i], other.sum[i]);
        }
      }
  }
  if (!writes) return;
  float *summary = reinterpret_cast<float *>(entries[2]) + at;
  const float page_rows = (float)(w + cnt);
  if (vectors) {
    *reinterpret_cast<uint4 *>(minimum) = *reinterpret_cast<const uint4 *>(low);
    *reinterpret_cast<uint4 *>(maximum) = *reinterpret_cast<const uint4 *>(high);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<float2 *>(summary)[i] = make_float2(sum[i].x / page_rows, sum[i].y / page_rows);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= n) break;
    minimum[i] = reinterpret_cast<const __nv_bfloat16 *>(low)[i];
    maximum[i] = reinterpret_cast<const __nv_bfloat16 *>(high)[i];
    summary[i] = (i % 2 ? sum[i / 2].y : sum[i / 2].x) / page_rows;
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
// Reads and writes are what bounds it, and close behind them its instructions. A thread
// takes as many codes at a time as make one vector of 16 bytes, so that neighbouring
// threads write whole sectors (16 codes a thread, half a sector a store: 285 us where 8 take
// 274, 262,144 rows of 8 heads of 128 in bf16; in fp32 half of them 293 and 4 codes 249).
// Where the next codes are follows from the last ones by additions: the divisions of a
// plain index took 339.
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
  int units;                  // of kN codes, in a plane of a row
  int step_rows, step_units;  // of kReadThreads units
  uint32_t head_magic;  // unit * head_magic / 2^32 is its head; 0: the unit itself is
  int32_t *status;
};

template <typename T, int kN>
__device__ __forceinline__ void write_values(T *to, const uint32_t (&codes)[(kN + 3) / 4],
                                             float scale) {
  if constexpr (kN == 1) {
    *to = from_f32<T>(decode4_f32(codes[0]).x * scale);
  } else {
    const float2 s = make_float2(scale, scale);
    alignas(16) T y[kN];
#pragma unroll
    for (int j = 0; j < kN; j += 4) {
      const float4 x = decode4_f32(codes[j / 4]);
      const float2 lo = pack_mul(make_float2(x.x, x.y), s);
      const float2 hi = pack_mul(make_float2(x.z, x.w), s);
      y[j] = from_f32<T>(lo.x);
      y[j + 1] = from_f32<T>(lo.y);
      y[j + 2] = from_f32<T>(hi.x);
      y[j + 3] = from_f32<T>(hi.y);
    }
    *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(y);
  }
}

template <typename T, int kN>
__global__ void __launch_bounds__(kReadThreads) read_quantized_kernel(ReadParams p) {
  constexpr int kWords = (kN + 3) / 4;
  __shared__ const unsigned char *records[2 * kReadRows];  // K's, then V's; NULL: zeros
  const int64_t row0 = (int64_t)blockIdx.x * kReadRows;
  const int rows = (int)min((int64_t)kReadRows, p.count - row0);
  if (threadIdx.x < rows) {
    const int64_t index = record_index(p.rows[row0 + threadIdx.x], p.page_size, p.page_shift,
                                       p.pool_blocks, p.status);
    records[threadIdx.x] = index < 0 ? nullptr : p.pool + index * p.record;
    records[rows + threadIdx.x] =
        index < 0 ? nullptr : p.pool + (index + p.page_size) * p.record;
  }
  __syncthreads();
  const int64_t E = (int64_t)p.kv_heads * p.head_dim;
  // a plane's results follow one another like the units do
  T *out = static_cast<T *>(p.out) + row0 * E + (int64_t)threadIdx.x * kN;
  const int64_t plane = (p.count - rows) * E;  // from the block's K rows' end to its V rows
  int r = threadIdx.x / p.units, c = threadIdx.x - r * p.units;
  while (r < 2 * rows) {
    uint32_t codes[kReadAhead][kWords];
    unsigned scale[kReadAhead];
    int rs[kReadAhead];
#pragma unroll
    for (int u = 0; u < kReadAhead; ++u) {
      rs[u] = r;
#pragma unroll
      for (int i = 0; i < kWords; ++i) codes[u][i] = 0;
      scale[u] = 127;
      const unsigned char *record = r < 2 * rows ? records[r] : nullptr;
      if (record != nullptr) {
        const unsigned char *from = record + (int64_t)c * kN;
        if constexpr (kN == 8) {
          const uint2 x = __ldg(reinterpret_cast<const uint2 *>(from));
          codes[u][0] = x.x;
          codes[u][1] = x.y;
        } else if constexpr (kN == 4) {
          codes[u][0] = __ldg(reinterpret_cast<const uint32_t *>(from));
        } else {
          codes[u][0] = __ldg(from);
        }
        const uint32_t head = p.head_magic ? __umulhi((uint32_t)c, p.head_magic) : (uint32_t)c;
        scale[u] = __ldg(record + E + head);
      }
      r += p.step_rows;
      c += p.step_units;
      if (c >= p.units) {
        c -= p.units;
        ++r;
      }
    }
#pragma unroll
    for (int u = 0; u < kReadAhead; ++u, out += kReadThreads * kN)
      if (rs[u] < 2 * rows)
        write_values<T, kN>(out + (rs[u] >= rows ? plane : 0), codes[u], scale_of(scale[u]));
  }
}

template <typename T, int kN> int launch_read(ReadParams p, cudaStream_t s) {
  p.units = (int)((int64_t)p.kv_heads * p.head_dim / kN);
  p.step_rows = kReadThreads / p.units;
  p.step_units = kReadThreads % p.units;
  // exact while units * (units of a head) stays below 2^32
  const uint32_t per_head = (uint32_t)(p.head_dim / kN);
  p.head_magic = per_head == 1 ? 0 : (uint32_t)((0x100000000ull + per_head - 1) / per_head);
  const unsigned grid = (unsigned)ceil_div(p.count, kReadRows);
  read_quantized_kernel<T, kN><<<grid, kReadThreads, 0, s>>>(p);
  return check_launch("read_quantized_kernel");
}
template <typename T> int launch_read(const ReadParams &p, cudaStream_t s) {
  const bool wide = reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  constexpr int kN = 16 / sizeof(T);  // one vector of results
  return wide && p.head_dim % kN == 0 ? launch_read<T, kN>(p, s) : launch_read<T, 1>(p, s);
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
  if ((int64_t)kv_heads * head_dim > (1 << 24))
    return set_error(HS_ERR_UNSUPPORTED, "append: heads too many");
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
  if (count > (int64_t)0x7fffffff * kReadRows || (int64_t)kv_heads * head_dim > (1 << 24))
    return set_error(HS_ERR_UNSUPPORTED, "read_quantized: rows or heads too many");
  ReadParams p{};
  p.pool = static_cast<const unsigned char *>(pool);
  p.pool_blocks = pool_blocks;
  p.rows = rows;
  p.count = count;
  p.out = out;
  p.kv_heads = kv_heads;
  p.head_dim = head_dim;
  p.page_size = page_size;
  p.page_shift = page_shift_of(page_size);
  p.record = record_bytes(kv_heads, head_dim);
  p.status = device_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case HS_FLOAT32: return launch_read<float>(p, s);
    case HS_FLOAT16: return launch_read<__half>(p, s);
    default: return launch_read<__nv_bfloat16>(p, s);
  }
}
