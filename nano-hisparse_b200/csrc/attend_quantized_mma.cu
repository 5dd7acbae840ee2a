// Decode attention over an 8-bit cache on tensor cores: head_dim a multiple of 16, heads
// that share their rows.
//
// A warp serves one KV head and up to 4 * kQuads of its query heads over units of 32
// rows: it copies its head's part of them (cp.async, 16 bytes a lane, into a ring of its
// own, two tiles of 16 rows ahead) and keeps its own maximum, sum and output. The heads of a
// block read neighbouring parts of the same rows and share one thing, the rows' scales: each
// of the warps in turn copies those of a unit for all of them, since 32 rows' scales are
// 32 requests of a few bytes for whoever reads them (a head's part of a row is one or
// two), and the number of requests is what bounds the reads. The ring of scales is deep enough that the
// warps hardly ever wait for one another. Keys are the M side of the products, 16 at a
// time:
//   S^T = K Q^T     m16n8k32 in e4m3: the codes go from ldmatrix to the tensor core as
//                   they are. Q is taken apart into e4m3 numbers, each a sixteenth of the
//                   one before it (q = q0 + q1 / 16 + ...): 2 parts hold bf16, 3 fp16 and
//                   6 fp32 exactly, since each part leaves at most 2^-4 of what it takes,
//                   but for elements below 2^-13 of the query's largest: those are off by up
//                   to 2^-21 of it in bf16 (e4m3 numbers end there), 2^-25 in fp16. Two
//                   parts of a query are neighbouring columns, whose sums meet in one lane.
//                   The products are exact and added in fp32 (measured: within
//                   2^-20 of the largest, as fp16 products are).
//   O^T += V^T P^T  m16n8k16 in fp16, which holds every e4m3 number. V through
//                   ldmatrix.trans, whose 16-bit unit is two neighbouring elements of a
//                   row: a byte permutation makes pairs of rows of each. P is the weight
//                   rounded to fp16 and, in the column beside it, 2^11 times what that left:
//                   22 bits together, and steps of 2^-35 where the first one's are of 2^-24
//                   (2^-43 of the largest weight; unscaled, 2^-32, the weights of a long flat
//                   tail behind one large row were all cut alike). Where two quads of bf16
//                   queries share the columns, what was left goes, as it is, through a
//                   second product into the same sums: half the registers for the output,
//                   as many products, 2^-32 of the largest weight a row where a result's
//                   own rounding is 2^-8. (A single product, 11 bits, took 39.5 us where this
//                   takes 40.7, 8 requests of 16,384 rows, 28/4 heads of 128, and 66.6 where
//                   this takes 72.8, 16 of 18,348, 12 heads of 256; but one result in twelve
//                   then differed from the weights' own by a step of bf16.)
// A weight is kept times 2^7 of the current maximum's, which is raised only when one would
// pass it by more than 2^8. A row whose V has the smallest scale (zeros) adds up to 2^115 to
// the sum: a sum that has passed 2^100 raises the maximum by 2^24, since 16,384 such rows of a
// warp would take it past fp32, and with it what other rows hold.
//
// 16 requests of 32,768 rows, 32/8 heads of 128, bf16 (959 MB) take 167 us: 5.7 TB/s, 88 % of
// a copy's rate. Rows in runs reach 5.8, single rows in any order 5.5. What else was measured
// of that call: scores in fp16, codes converted, 213; scales copied by each warp for itself
// 197, since 32 of its 96 requests a tile were for one byte; whole records copied by one
// warp of the block 208, by all warps 208; boxes of tiled copies 185 (75 clocks of the copy
// engine a box); fragments straight from global memory 250. With 7 query heads a KV head the
// warps' instructions are level with the reads (8 requests of 16,384 rows, 4 KV heads: 38 to
// 41 us, floor 20.7), with more of them ahead.
#include <type_traits>

#include "attend_quantized.cuh"

namespace hs {
namespace {

constexpr int kMmaWarps = 8, kMmaThreads = 32 * kMmaWarps;
constexpr int kMmaRows = 16;     // rows of a tile, a stage of the ring
constexpr int kUnitRows = 32;    // two tiles: a lane has the number of one of their rows
constexpr int kStages = 3;       // the two tiles after the one that is worked on are on their way
constexpr int kSlots = 8;        // units whose scales are kept
constexpr int kAhead = 2;        // units that scales are copied ahead
// A unit's scales of one plane: 4 bytes a row where all heads' are in one word, else the
// one or two 16-byte chunks of a row that have the block's heads
constexpr int kScaleRoom = 16 * 1024;  // of all rings of scales: 8 of words or 1 of two chunks
constexpr float kWeightLift = 7.f, kRaise = 15.f;  // lifted weights stay below 2^kRaise
constexpr float kLeftLift = 2048.f;                // of what a weight's rounding to fp16 left
constexpr float kSumShare = 0x1p-96f, kSumStep = 24.f;  // of a sum to compare with kRaise
constexpr float kNothing = 1e38f;                  // base of a query that has seen nothing

// parts of a query element
template <typename T> constexpr int kQueryParts = 2;
template <> constexpr int kQueryParts<__half> = 3;
template <> constexpr int kQueryParts<float> = 6;

template <typename T, int kDim, int kQuads> struct MmaShape {
  static constexpr int query_tiles = (kQueryParts<T> + 1) / 2;  // of 8 columns, for each quad
  static constexpr bool paired = std::is_same<T, __nv_bfloat16>::value && kQuads > 1;
  static constexpr int output_tiles = paired ? kQuads / 2 : kQuads;
  static constexpr int plane = kMmaRows * kDim;
  static constexpr int stage = 2 * plane;  // K, V
  static constexpr int queries = 4 * kQuads;
  static constexpr int ring = kStages * stage;
  // a warp's results at the end, in the place of its ring: its queries' elements (the rows'
  // pitch keeps the stores of four queries in different banks) and statistics, and in the
  // first slice's the statistics of all slices together
  static constexpr int pitch = kDim + 16, result = queries * pitch * 4;
  static_assert(result + 2 * queries * (int)sizeof(float2) <= ring, "the results fit a ring");
  static constexpr int rings = kMmaWarps * ring;
  // the rings of scales, and their barriers: for each slice of the warps full and free
  static constexpr size_t bytes = rings + kScaleRoom + kMmaWarps * 2 * kSlots * sizeof(uint64_t);
  // blocks on an SM: two where the output and the queries leave the registers for it
  static constexpr int resident =
      kDim / 4 * output_tiles + kDim / 16 * kQuads * query_tiles <= 64 && kDim <= 128 ? 2 : 1;
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
__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// Place of 16-byte chunk c of row r of a tile: rows of 128 bytes (64 where kDim is 64),
// panel after panel, swizzled so that the eight rows of an ldmatrix are in different
// banks. Chunk c + i of a row, c < 2 and i even, is at the place of c changed by
// tile_chunk.
template <int kDim> __device__ __forceinline__ uint32_t tile_place(int r, int c) {
  if constexpr (kDim == 64) return r * 64 + ((c ^ (r >> 1 & 3)) << 4);
  return (c >> 3) * (kMmaRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}
template <int kDim> __device__ __forceinline__ uint32_t tile_chunk(uint32_t place, int i) {
  return (place ^ (i & 7) << 4) + (i >> 3) * (kMmaRows * 128);
}
// Arrives on `bar` once this thread's copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_addr(bar))
               : "memory");
}
// The parts of four query elements, two for each tile of columns
template <typename T, int kTiles>
__device__ __forceinline__ void split_query(float4 x, uint32_t (&codes)[2 * kTiles]) {
#pragma unroll
  for (int part = 0; part < 2 * kTiles; ++part) {
    codes[part] = part < kQueryParts<T> ? encode4(x.x, x.y, x.z, x.w) : 0u;
    const float4 y = decode4_f32(codes[part]);
    x = make_float4((x.x - y.x) * 16.f, (x.y - y.y) * 16.f, (x.z - y.z) * 16.f,
                    (x.w - y.w) * 16.f);
  }
}
// Four query elements as they lie in memory
template <typename T> struct Raw4 {
  uint2 raw;
  __device__ __forceinline__ void load(const T *from) {
    raw = __ldg(reinterpret_cast<const uint2 *>(from));
  }
  __device__ __forceinline__ void clear() { raw = make_uint2(0u, 0u); }
  __device__ __forceinline__ float4 get() const {
    const T *x = reinterpret_cast<const T *>(&raw);
    return make_float4(to_f32(x[0]), to_f32(x[1]), to_f32(x[2]), to_f32(x[3]));
  }
};
template <> struct Raw4<float> {
  float4 raw;
  __device__ __forceinline__ void load(const float *from) {
    raw = __ldg(reinterpret_cast<const float4 *>(from));
  }
  __device__ __forceinline__ void clear() { raw = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ float4 get() const { return raw; }
};
// A query's results of n <= kMost parts of its rows, joined: stat(i) is part i's maximum and
// sum, element(i) a pair of its elements. A part that saw nothing has left zeros.
struct Joined {
  float top, sum;
  float2 x;
};
template <int kMost, typename Stat, typename Element>
__device__ __forceinline__ Joined join(int n, Stat stat, Element element) {
  float2 s[kMost], x[kMost];
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    s[i] = i < n ? stat(i) : make_float2(-kNothing, 0.f);
    x[i] = i < n ? element(i) : make_float2(0.f, 0.f);
  }
  Joined all{s[0].x, 0.f, make_float2(0.f, 0.f)};
#pragma unroll
  for (int i = 1; i < kMost; ++i) all.top = fmaxf(all.top, s[i].x);
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const float w = s[i].y == 0.f ? 0.f : quant_exp2(s[i].x - all.top);
    all.sum = fmaf(w, s[i].y, all.sum);
    all.x.x = fmaf(w, x[i].x, all.x.x);
    all.x.y = fmaf(w, x[i].y, all.x.y);
  }
  return all;
}

template <typename T, int kDim, int kQuads>
__global__ void __launch_bounds__(kMmaThreads, MmaShape<T, kDim, kQuads>::resident)
    quant_mma_kernel(QuantAttendParams p, int heads_of_block, int head_places, bool cluster) {
  using Shape = MmaShape<T, kDim, kQuads>;
  constexpr int kChunks = kDim / 16, kQueries = Shape::queries;
  constexpr int kQueryTiles = Shape::query_tiles, kOutputTiles = Shape::output_tiles;
  constexpr bool kPaired = Shape::paired;
  constexpr uint32_t kNone = 0xffffffffu;
  extern __shared__ __align__(128) unsigned char smem[];
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int lane = threadIdx.x & 31, D = p.head_dim;
  const int warp = __shfl_sync(kFullMask, threadIdx.x >> 5, 0);
  const int split = blockIdx.x, b = blockIdx.z;
  const int chunks = (p.groups + kQueries - 1) / kQueries;  // of a KV head's query heads
  const int group = blockIdx.y / chunks, chunk = blockIdx.y - group * chunks;
  const int place_bits = __popc(head_places - 1);  // head_places is a power of two
  const int slices = kMmaWarps >> place_bits;      // warps that share a head's rows
  const int place = warp & (head_places - 1), slice = warp >> place_bits;
  const int kh = group * heads_of_block + place;
  const bool here = place < heads_of_block && kh < p.kv_heads;
  const int h0 = kh * p.groups + chunk * kQueries;
  const int hn = here ? min(kQueries, p.groups - chunk * kQueries) : 0;  // query heads

  // Q is read first and used after the first copies are on their way. A column lane / 4 of
  // a tile is query head lane / 8 of a quad, part lane / 4 % 2; of every 16 elements the
  // lane has those at 4 * (lane % 4) on. It reads and takes apart every other 16 elements,
  // which its neighbour 4 lanes on has too, and gives it the parts that are its own.
  const bool odd = lane & 4;
  Raw4<T> raw[kQuads][kChunks / 2];
#pragma unroll
  for (int n = 0; n < kQuads; ++n) {
    const int g = n * 4 + lane / 8;
    const T *from = static_cast<const T *>(p.query) + (int64_t)b * p.q_batch_stride +
                    (int64_t)(h0 + g) * D + lane % 4 * 4;
#pragma unroll
    for (int c = 0; c < kChunks / 2; ++c) {
      const int at = (2 * c + odd) * 16;
      if (g < hn && at < D) raw[n][c].load(from + at);
      else raw[n][c].clear();
    }
  }

  // this warp's units: first, first + slices, ... < last
  const int valid = (int)quant_rows(p, b), units = (valid + kUnitRows - 1) / kUnitRows;
  const int share = units / p.splits, rest = units - share * p.splits;
  const int first = share * split + rest * split / p.splits + slice;
  const int last = here ? share * (split + 1) + rest * (split + 1) / p.splits : 0;

  // A lane has the row number of one row of a unit, read one unit before its copies.
  const int64_t *rows = p.rows + b * p.rows_batch_stride;
  const auto look = [&](int unit) -> int64_t {
    const unsigned at = (unsigned)unit * kUnitRows + lane;
    return unit < last && at < (unsigned)valid ? __ldg(rows + at) : -1;
  };
  // The index of its K record; the launch has checked that all of them fit 32 bits.
  const int64_t pool_rows = p.pool_blocks * p.page_size;
  const auto record_of = [&](int64_t row) -> uint32_t {
    if (row < 0) return kNone;
    if (row >= pool_rows) {
      flag(p.status, HS_DEV_ROW_OUT_OF_RANGE);
      return kNone;
    }
    const uint32_t r = (uint32_t)row, P = (uint32_t)p.page_size;
    return r + (p.page_shift >= 0 ? r & ~(P - 1) : r / P * P);  // block * 2 P + within
  };
  // scales: a ring for each slice of the warps
  const int width = p.kv_heads <= 4 ? 4 : (group * heads_of_block & 15) + heads_of_block > 16 ? 32 : 16;
  unsigned char *scales = smem + Shape::rings + slice * (kSlots * 2 * kUnitRows) * width;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + Shape::rings + kScaleRoom) +
                   slice * 2 * kSlots, *free = full + kSlots;
  const int sharing = min(head_places, min(heads_of_block, p.kv_heads - group * heads_of_block));
  if (place == 0 && lane < 2 * kSlots) {
    mbar_init(&full[lane], lane < kSlots ? 32 : sharing);  // free follows full
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();
  const uint32_t record = (uint32_t)p.record, ring = smem_addr(smem) + warp * Shape::ring;
  const int c16 = lane % kChunks * 16;
  const int copied = c16 < D ? 16 : 0;  // chunks past head_dim are zeros
  const int64_t v_plane = (int64_t)p.page_size * p.record;
  const unsigned char *chunk_of = p.pool + (copied ? (int64_t)kh * D + c16 : 0);
  const int scale0 = width == 4 ? 0 : group * heads_of_block & ~15;  // the first head's of a slot
  const unsigned char *scale_of_row = p.pool + (int64_t)p.kv_heads * D + scale0;
  const auto copy_tile = [&](uint32_t index, int half, int stage) {
    constexpr int together = 32 / kChunks;  // rows of a step
#pragma unroll
    for (int i = 0; i < kMmaRows / together; ++i) {
      const uint32_t at =
          __shfl_sync(kFullMask, index, half * kMmaRows + i * together + lane / kChunks);
      const int bytes = at != kNone ? copied : 0;
      const unsigned char *src = chunk_of + (uint64_t)(at != kNone ? at : 0u) * record;
      const uint32_t dst = ring + stage * Shape::stage +
                           tile_place<kDim>(i * together + lane / kChunks, lane % kChunks);
      copy16(dst, src, bytes);
      copy16(dst + Shape::plane, src + v_plane, bytes);
    }
  };
  // The scales of the i-th unit of this slice, a row a lane, into slot i % kSlots; i counts
  // the units that the warps of the slice have in common.
  bool ok = true;
  const auto copy_scales = [&](int i, uint32_t at) {
    if (i >= kSlots) {
      ok = __all_sync(kFullMask, wait_phase(&free[i % kSlots], (i / kSlots - 1) & 1, p.status));
      if (!ok) return;
    }
    const unsigned char *src = scale_of_row + (uint64_t)(at != kNone ? at : 0u) * record;
    const uint32_t dst = smem_addr(scales) + ((i % kSlots) * 2 * kUnitRows + lane) * width;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      if (width == 4) {
        copy4(dst + plane * kUnitRows * 4, src + plane * v_plane, at != kNone ? 4 : 0);
      } else {
        copy16(dst + plane * kUnitRows * width, src + plane * v_plane, at != kNone ? 16 : 0);
        if (width == 32)
          copy16(dst + plane * kUnitRows * width + 16, src + plane * v_plane + 16,
                 at != kNone ? 16 : 0);
      }
    }
    copies_arrive(&full[i % kSlots]);
  };
  uint32_t index = kNone;   // of the unit whose tiles are copied next
  int64_t next = look(first), later = look(first + slices);  // row numbers of the units after it
  int to = 0;               // stage of the next copy
  const auto copy_half = [&](int unit, int half) {
    if (unit < last) {
      if (half == 0) {
        index = record_of(next);
        next = later;
        later = look(unit + 2 * slices);
      }
      copy_tile(index, half, to);
    }
    to = to == kStages - 1 ? 0 : to + 1;
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  static_assert(kAhead == 2, "next and later");
  if (place == 0 && first < last) copy_scales(0, record_of(next));
  if (place == (sharing > 1) && first + slices < last) copy_scales(1, record_of(later));
  copy_half(first, 0);
  copy_half(first, 1);

  uint32_t q[kQuads][kQueryTiles][kChunks];
  float factor[kQuads];  // of the scores of query head lane % 4
#pragma unroll
  for (int n = 0; n < kQuads; ++n) {
    float largest = 0.f;
#pragma unroll
    for (int c = 0; c < kChunks / 2; ++c) {
      const float4 x = raw[n][c].get();
      largest = fmaxf(fmaxf(largest, fmaxf(fabsf(x.x), fabsf(x.y))),
                      fmaxf(fabsf(x.z), fabsf(x.w)));
    }
#pragma unroll
    for (int i = 1; i < 8; i <<= 1)
      largest = fmaxf(largest, __shfl_xor_sync(kFullMask, largest, i));
    // to between 128 and 256: what is 2^13 times smaller is still a normal e4m3 number. An
    // infinity leaves NaN, as its scores are
    const int e = (__float_as_int(largest) >> 23) - 127 - 7;
    const float scale = largest > 0.f ? power_of_two(max(-126, min(127, -e))) : 1.f;
    const bool finite = largest < INFINITY;
#pragma unroll
    for (int c = 0; c < kChunks / 2; ++c) {
      const float4 x = raw[n][c].get();
      uint32_t codes[2 * kQueryTiles];
      split_query<T, kQueryTiles>(
          make_float4(x.x * scale, x.y * scale, x.z * scale, x.w * scale), codes);
#pragma unroll
      for (int t = 0; t < kQueryTiles; ++t) {
        const uint32_t even_part = finite ? codes[2 * t] : 0x7f7f7f7fu;
        const uint32_t odd_part = finite ? codes[2 * t + 1] : 0x7f7f7f7fu;
        const uint32_t own = odd ? odd_part : even_part;
        const uint32_t other = __shfl_xor_sync(kFullMask, odd ? even_part : odd_part, 4);
        q[n][t][2 * c] = odd ? other : own;
        q[n][t][2 * c + 1] = odd ? own : other;
      }
    }
    factor[n] = __shfl_sync(kFullMask, p.scale_log2 / scale, lane % 4 * 8);
  }

  // base: lift less the maximum, added to a score before its power is taken
  float base[kQuads], l[kQuads], o[kOutputTiles][kChunks][4];
#pragma unroll
  for (int n = 0; n < kQuads; ++n) {
    base[n] = kNothing;
    l[n] = 0.f;
  }
#pragma unroll
  for (int n = 0; n < kOutputTiles; ++n)
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][c][i] = 0.f;
  // ldmatrix: matrix lane / 8 has rows (lane / 8 % 2) * 8 on, chunk lane / 16
  const uint32_t matrix = ring + tile_place<kDim>(lane & 15, lane / 16);
  const unsigned char *scale_byte = scales + lane / 4 * width + (kh - scale0);
  int stage = 0, count = 0;
  // whose turn the scales of the unit kAhead units on are
  int turn = sharing > 2 ? 2 : 0;
  for (int unit = first; unit < last && ok; unit += slices, ++count) {
    // row numbers of unit + 2 * slices are in `next` until the copies below move on
    if (turn == place && unit + kAhead * slices < last) {
      copy_scales(count + kAhead, record_of(later));
      if (!ok) break;
    }
    turn = turn == sharing - 1 ? 0 : turn + 1;
    const int slot = count % kSlots;
    ok = __all_sync(kFullMask, wait_phase(&full[slot], count / kSlots & 1, p.status));
    if (!ok) break;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 2) : "memory");
      __syncwarp();
      copy_half(unit + slices, half);
      const uint32_t tile = matrix + stage * Shape::stage;
      const unsigned char *bytes = scale_byte + (slot * 2 * kUnitRows + half * kMmaRows) * width;
      stage = stage == kStages - 1 ? 0 : stage + 1;
      if (unit * kUnitRows + half * kMmaRows >= valid) continue;  // the last unit's second half
      // ---- S^T: rows lane / 4 and lane / 4 + 8, query head lane % 4 of each quad
      float s[kQuads][kQueryTiles][4];
#pragma unroll
      for (int n = 0; n < kQuads; ++n)
#pragma unroll
        for (int t = 0; t < kQueryTiles; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][t][i] = 0.f;
#pragma unroll
      for (int c = 0; c < kChunks; c += 2) {
        uint32_t k[4];
        ldmatrix4(k, tile_chunk<kDim>(tile, c));
#pragma unroll
        for (int n = 0; n < kQuads; ++n)
#pragma unroll
          for (int t = 0; t < kQueryTiles; ++t)
            mma_e4m3(s[n][t], k, q[n][t][c], q[n][t][c + 1]);
      }
      // a row that is not seen has zeros in the place of its scale, which is never 0
      const unsigned ek[2] = {bytes[0], bytes[8 * width]};
      const unsigned ev[2] = {bytes[kUnitRows * width], bytes[(kUnitRows + 8) * width]};
      float k_scale[2], v_exponent[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        k_scale[r] = scale_of(ek[r]);
        // byte - 127 as a float: the byte under 2^23's exponent
        v_exponent[r] = __uint_as_float(0x4b000000u | ev[r]) - (8388608.f + 127.f);
      }
      // exponents of the weights: x in the sum, y in the output, lifted
      float x[kQuads][2], y[kQuads][2], lifted[kQuads][2], top_lifted = -INFINITY;
#pragma unroll
      for (int n = 0; n < kQuads; ++n) {
        top_lifted = fmaxf(top_lifted, l[n] * kSumShare);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float dot = 0.f;
#pragma unroll
          for (int t = kQueryTiles - 1; t >= 0; --t)
            dot = fmaf(dot, 1.f / 256.f, fmaf(s[n][t][2 * r + 1], 1.f / 16.f, s[n][t][2 * r]));
          // chosen, not added: the product is NaN for a query that is not finite
          x[n][r] = ek[r] != 0 ? dot * (k_scale[r] * factor[n]) : -INFINITY;
          y[n][r] = x[n][r] + v_exponent[r];
          lifted[n][r] = y[n][r] + base[n];
          top_lifted = fmaxf(top_lifted, lifted[n][r]);
        }
      }
      if (__any_sync(kFullMask, top_lifted > kRaise)) {
        float f[kQuads];
#pragma unroll
        for (int n = 0; n < kQuads; ++n) {
          float top = fmaxf(y[n][0], y[n][1]);
          if (l[n] * kSumShare > kRaise) top = fmaxf(top, kWeightLift + kSumStep - base[n]);
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, i));
          // (a base of kNothing makes f 0)
          const float to_base = fminf(base[n], kWeightLift - top);
          f[n] = quant_exp2(to_base - base[n]);
          base[n] = to_base;
          l[n] *= f[n];
#pragma unroll
          for (int r = 0; r < 2; ++r) lifted[n][r] = y[n][r] + to_base;
        }
#pragma unroll
        for (int n = 0; n < kOutputTiles; ++n)
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][c][i] *= kPaired ? f[2 * n + (i & 1)] : f[n];
      }
#pragma unroll
      for (int n = 0; n < kQuads; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          l[n] += quant_exp2(x[n][r] + base[n]);
          y[n][r] = quant_exp2(lifted[n][r]);
        }
      uint32_t w[kOutputTiles][2], left[kOutputTiles][2];  // left: what rounding left, if paired
#pragma unroll
      for (int n = 0; n < kOutputTiles; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (kPaired) {
            const float even = y[2 * n][r], odd = y[2 * n + 1][r];
            const __half2 rounded = __floats2half2_rn(even, odd);
            w[n][r] = transpose8(*reinterpret_cast<const uint32_t *>(&rounded));
            left[n][r] = transpose8(
                pack_half(even - __low2float(rounded), odd - __high2float(rounded)));
          } else {
            const __half rounded = __float2half_rn(y[n][r]);
            w[n][r] = transpose8(
                pack_half(y[n][r], (y[n][r] - __half2float(rounded)) * kLeftLift));
          }
        }
      // ---- O^T: elements 16 c + 2 * (lane / 4) + 0, 1, columns 2 * (lane % 4) + 0, 1
#pragma unroll
      for (int c = 0; c < kChunks; c += 2) {
        uint32_t v[4];
        ldmatrix4_trans(v, tile_chunk<kDim>(tile, c) + Shape::plane);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint2 lo = decode4(__byte_perm(v[2 * u], 0, 0x3120));
          const uint2 hi = decode4(__byte_perm(v[2 * u + 1], 0, 0x3120));
#pragma unroll
          for (int n = 0; n < kOutputTiles; ++n) {
            mma_f16(o[n][c + u], lo.x, lo.y, hi.x, hi.y, w[n][0], w[n][1]);
            if constexpr (kPaired)
              mma_f16(o[n][c + u], lo.x, lo.y, hi.x, hi.y, left[n][0], left[n][1]);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&free[slot]);
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");

  // ---- results: out = o / l, in the join's terms o 2^-kSumLift / l 2^kSumLift ------------
  const int64_t part0 = quant_part(p, p.phase, b, 0, split);
  const int pad = quant_pad(D);
  const auto write = [&](int h, int d, float top, float sum, float2 x) {
    if (p.out != nullptr) {
      const float inv = sum > 0.f || sum != sum ? kSumScale / sum : 0.f;
      T *out = static_cast<T *>(p.out) + ((int64_t)b * p.q_heads + h) * D + d;
      out[0] = from_f32<T>(x.x * inv);
      out[1] = from_f32<T>(x.y * inv);
    } else {
      const int64_t part = part0 + (unsigned)(h * p.splits);
      if (d == 0) p.stats[part] = make_float4(top, 0.f, sum, 0.f);
      *reinterpret_cast<float2 *>(p.partials + part * pad + d) = x;
    }
  };
  // elements 16 c + 2 * (lane / 4) + 0, 1 of query head lane % 4 of quad n
  const auto result = [&](int n, int c) {
    const float(&x)[4] = o[kPaired ? n / 2 : n][c];
    const float2 sum = kPaired ? make_float2(x[n & 1], x[2 + (n & 1)])
                               : make_float2(fmaf(x[1], 1.f / kLeftLift, x[0]),
                                             fmaf(x[3], 1.f / kLeftLift, x[2]));
    return make_float2(sum.x * (1.f / kSumScale), sum.y * (1.f / kSumScale));
  };
#pragma unroll
  for (int n = 0; n < kQuads; ++n)
#pragma unroll
    for (int i = 4; i < 32; i <<= 1) l[n] += __shfl_xor_sync(kFullMask, l[n], i);
  if (slices == 1 && !cluster) {
#pragma unroll
    for (int n = 0; n < kQuads; ++n)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int g = n * 4 + lane % 4, d = c * 16 + lane / 4 * 2;
        if (g < hn && d < D) write(h0 + g, d, -base[n], l[n], result(n, c));
      }
    return;
  }
  // The results of the slices meet in shared memory, then those of the splits in a cluster:
  // a thread takes pairs of elements and reads the statistics beside them. Every thread of
  // the cluster comes to both of its barriers.
  constexpr int kPitch = Shape::pitch, kPairs = kDim / 2, kStep = kMmaThreads / kPairs;
  // of warp w: elements, statistics and, of the first slice's, all slices' statistics
  const auto elements = [&](int w) { return reinterpret_cast<float *>(smem + w * Shape::ring); };
  const auto stats = [&](int w, int of) {
    return reinterpret_cast<float2 *>(smem + w * Shape::ring + Shape::result) + of * kQueries;
  };
#pragma unroll
  for (int n = 0; n < kQuads; ++n) {
    float *to_query = elements(warp) + (n * 4 + lane % 4) * kPitch;
    if (lane < 4) stats(warp, 0)[n * 4 + lane] = make_float2(-base[n], l[n]);
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      *reinterpret_cast<float2 *>(to_query + c * 16 + lane / 4 * 2) = result(n, c);
  }
  const int queries = min(kQueries, p.groups - chunk * kQueries);
  const int d = threadIdx.x % kPairs * 2, first_query = threadIdx.x / kPairs;
  const int all = d < D ? sharing * kQueries : 0;
  const auto join_slices = [&](auto n) {
    constexpr int kParts = decltype(n)::value;
    for (int i = first_query; i < all; i += kStep) {
      const int head = i / kQueries, g = i % kQueries;
      if (g >= queries) continue;
      const Joined x = join<kParts>(
          kParts, [&](int k) { return stats(k * head_places + head, 0)[g]; },
          [&](int k) {
            return *reinterpret_cast<const float2 *>(elements(k * head_places + head) +
                                                     g * kPitch + d);
          });
      if (!cluster) {
        write((group * heads_of_block + head) * p.groups + chunk * kQueries + g, d, x.top, x.sum,
              x.x);
      } else {  // read by this thread alone so far
        *reinterpret_cast<float2 *>(elements(head) + g * kPitch + d) = x.x;
        if (d == 0) stats(head, 1)[g] = make_float2(x.top, x.sum);
      }
    }
  };
  static_assert(kMmaWarps == 8, "the numbers of slices");
  if (slices > 1) {
    __syncthreads();
    if (slices == 2) join_slices(std::integral_constant<int, 2>());
    else if (slices == 4) join_slices(std::integral_constant<int, 4>());
    else join_slices(std::integral_constant<int, 8>());
  }
  if (!cluster) return;
  cluster_barrier();
  for (int i = split * kStep + first_query; i < all; i += p.splits * kStep) {
    const int head = i / kQueries, g = i % kQueries;
    if (g >= queries) continue;
    const Joined x = join<kClusterSplits>(
        p.splits, [&](int k) { return *map_rank(stats(head, slices > 1 ? 1 : 0) + g, k); },
        [&](int k) {
          return *reinterpret_cast<const float2 *>(
              map_rank(elements(head) + g * kPitch + d, k));
        });
    write((group * heads_of_block + head) * p.groups + chunk * kQueries + g, d, x.top, x.sum, x.x);
  }
  cluster_barrier();  // the others may still read this block's results
}

// Quads of a warp at most: what the registers hold
template <typename T, int kDim>
constexpr int kMostQuads = kDim == 64 || std::is_same<T, __nv_bfloat16>::value ? 4
                           : std::is_same<T, __half>::value                    ? 2
                                                                               : 256 / kDim;

template <typename T, int kDim, int kQuads>
int launch(const QuantAttendParams &p, const QuantMmaGrid &g, cudaStream_t s) {
  auto kernel = quant_mma_kernel<T, kDim, kQuads>;
  const size_t bytes = MmaShape<T, kDim, kQuads>::bytes;
  if (int e = reserve_smem(reinterpret_cast<const void *>(kernel), bytes, "attend_quantized"))
    return e;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)p.splits, (unsigned)(g.groups * g.chunks), (unsigned)p.batch);
  config.blockDim = dim3(kMmaThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = s;
  // the splits of a request are one cluster where they write its output
  const bool cluster = p.out != nullptr && p.splits > 1;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = (unsigned)p.splits;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = cluster ? 1 : 0;
  cudaLaunchKernelEx(&config, kernel, p, g.heads, g.places, cluster);
  return check_launch("quant_mma_kernel");
}
// Calls f with kDim and kQuads for a KV head's `per` query heads.
template <typename T, int kDim, typename F> auto with_quads(int per, F f) {
  constexpr int most = kMostQuads<T, kDim>;
  if constexpr (most >= 4)
    if (per > 8) return f(std::integral_constant<int, kDim>(), std::integral_constant<int, 4>());
  if constexpr (most >= 2)
    if (per > 4) return f(std::integral_constant<int, kDim>(), std::integral_constant<int, 2>());
  return f(std::integral_constant<int, kDim>(), std::integral_constant<int, 1>());
}
template <typename T, typename F> auto with_shape(int per, int head_dim, F f) {
  if (head_dim <= 64) return with_quads<T, 64>(per, f);
  if (head_dim <= 128) return with_quads<T, 128>(per, f);
  return with_quads<T, 256>(per, f);
}
template <typename T> QuantMmaGrid grid_of(int per, int kv_heads, int head_dim) {
  QuantMmaGrid g = with_shape<T>(per, head_dim, [](auto dim, auto quads) {
    QuantMmaGrid shape{};
    shape.queries = 4 * quads();
    shape.resident = MmaShape<T, dim(), quads()>::resident;
    return shape;
  });
  g.chunks = (per + g.queries - 1) / g.queries;
  g.groups = (kv_heads + kMmaWarps - 1) / kMmaWarps;
  g.heads = (kv_heads + g.groups - 1) / g.groups;
  g.groups = (kv_heads + g.heads - 1) / g.heads;
  for (g.places = 1; g.places < g.heads; g.places <<= 1) {}
  g.slices = kMmaWarps / g.places;
  return g;
}
template <typename T> int launch(const QuantAttendParams &p, cudaStream_t s) {
  return with_shape<T>(p.groups, p.head_dim, [&](auto dim, auto quads) {
    return launch<T, dim(), quads()>(p, grid_of<T>(p.groups, p.kv_heads, p.head_dim), s);
  });
}

}  // namespace

QuantMmaGrid quant_mma_grid(int dtype, int q_heads, int kv_heads, int head_dim) {
  const int per = q_heads / kv_heads;
  switch (dtype) {
    case HS_FLOAT32: return grid_of<float>(per, kv_heads, head_dim);
    case HS_FLOAT16: return grid_of<__half>(per, kv_heads, head_dim);
    default: return grid_of<__nv_bfloat16>(per, kv_heads, head_dim);
  }
}

int launch_quant_mma(const QuantAttendParams &p, int dtype, cudaStream_t s) {
  switch (dtype) {
    case HS_FLOAT32: return launch<float>(p, s);
    case HS_FLOAT16: return launch<__half>(p, s);
    default: return launch<__nv_bfloat16>(p, s);
  }
}

}  // namespace hs
