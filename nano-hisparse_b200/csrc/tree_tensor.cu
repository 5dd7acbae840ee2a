// Tree attention on the fifth-generation tensor cores: 16-bit types, head_dim <= 128.
//
// A block has one SM and up to 256 query rows as two streams of 128 (a stream is
// the M = 128 tile of tcgen05.mma, its rows the TMEM lanes). With more than 128
// rows stream w owns rows 128 w .. and both work on every block of 64 keys; with
// fewer, both own the same rows and take the key blocks in turn, so that one
// stream's softmax runs beside the other's products, and join at the end. 13 warps:
//   warps 0-3, 4-7  softmax of stream 0, 1: a thread has one query row. Scores
//                   from TMEM, P = exp2(s - m) rounded to the 16-bit type back to
//                   TMEM. The maximum is raised only when a score passes it by
//                   more than 8 (a factor of 256, inside fp16's range), so the
//                   output, which stays in TMEM, is rescaled rarely.
//   warps 8-11      copy key blocks, 16 bytes a thread with cp.async, into a ring
//                   of stages in the 128-byte-swizzled layout of the descriptors:
//                   rows are scattered over the pool, so there is no tile for the
//                   TMA engine, and a row's slice of one KV head is 256 bytes.
//   warp 12         one thread issues the products:
//                     S = Q K^T  both operands in shared memory, K-major
//                     O += P V   P in TMEM, V in shared memory, MN-major (as
//                                stored: a key's elements are adjacent)
// Scores of the next block are issued before the output of this one, so the
// tensor pipe and the softmax overlap. What bounds it: up to about 50 nodes the
// reads of K and V, beyond that the exponentials (16 a clock on an SM).
//
// TMEM columns of a stream: O 0..127, S 128..191, P (two buffers) 192..255.
// Every wait is bounded; one that runs out sets HS_DEV_WAIT_TIMEOUT, ends its
// warp's loop, and so lets every other wait run out.
#include <type_traits>

#include "tree.cuh"

namespace hs {
namespace {

constexpr int kSoftmaxWarps = 8, kLoadWarps = 4;
constexpr int kLoadThreads = 32 * kLoadWarps;
constexpr int kTensorThreads = 32 * (kSoftmaxWarps + kLoadWarps + 1);
constexpr int kTile = 128;     // query rows of a stream
constexpr int kKeys = 64;      // keys of a block
constexpr int kColumnsS = 128, kColumnsP = 192, kStreamColumns = 256;

// Shared memory of a block. kDim: head_dim rounded up to 64 or 128, the rest zero.
// Operands are panels of 64 elements (128 bytes) a row, 8 rows to the swizzle atom.
template <int kDim> struct TensorShape {
  static constexpr int panels = kDim / 64;
  static constexpr int q_bytes = kTile * kDim * 2;       // of one stream
  static constexpr int plane_bytes = kKeys * kDim * 2;   // K or V of a stage
  static constexpr int stages = kDim == 64 ? 8 : 5;
  static constexpr int ahead = kDim == 64 ? 4 : 2;       // stages left in flight
  static constexpr int ring = 2 * q_bytes;
  static constexpr int bytes = ring + stages * 2 * plane_bytes;
  static constexpr size_t dynamic = bytes + 1024;        // alignment to a swizzle atom
  static constexpr int join_pitch = kDim + 1;            // floats; the streams' join
  // The first product of a stream's next block is issued two blocks ahead of the
  // one whose stage is waited for; stages copied but not yet announced come on top.
  static_assert(ahead <= stages - 3, "the loader would wait for blocks it has not announced");
  static_assert(kTile * join_pitch * 4 <= stages * 2 * plane_bytes, "join fits the ring");
};

// 32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_load32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, "
               "%9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
               "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
                 "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
                 "=r"(r[30]), "=r"(r[31])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, "
               "%8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
               "%23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
               ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
                 "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
                 "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
                 "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
                 "r"(r[31])
               : "memory");
}
// The loads are done; the registers pass through so that no use moves ahead of it.
__device__ __forceinline__ void tmem_load_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_store_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ void fence_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
}
// Arrives on `bar` once the products issued so far are done.
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(
                   smem_addr(bar))
               : "memory");
}
// D = A B (+ D), both operands in shared memory
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                           bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// A in TMEM
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                         bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Shared-memory descriptor, 128-byte swizzle: `group` is the distance of panels
// (used by MN-major operands that span several), `atom` that of 8-row atoms.
__device__ __forceinline__ uint64_t descriptor(uint32_t addr, uint32_t group, uint32_t atom) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(group >> 4) << 16 |
         (uint64_t)(atom >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// Instruction descriptor: fp32 accumulator, M = 128, n columns; b_mn: B is MN-major
template <typename T> __device__ __forceinline__ uint32_t instruction(int n, bool b_mn) {
  constexpr uint32_t type = std::is_same<T, __half>::value ? 0 : 1;  // fp16, bf16
  return 1u << 4 | type << 7 | type << 10 | (uint32_t)b_mn << 16 | (uint32_t)(n >> 3) << 17 |
         (uint32_t)(kTile >> 4) << 24;
}
// Place of 16-byte chunk c of row r in a panelled, swizzled operand of `rows` rows
__device__ __forceinline__ uint32_t place(int r, int c, int rows) {
  return (uint32_t)((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

struct TensorBarriers {
  uint64_t kv_full[8], kv_free[8];
  uint64_t s_full[2], s_free[2];        // by stream
  uint64_t p_full[2][2], pv_done[2][2];  // by stream and P buffer
};

template <typename T, int kDim>
__global__ void __launch_bounds__(kTensorThreads, 1) tree_tensor_kernel(TreeParams p) {
  using Shape = TensorShape<kDim>;
  extern __shared__ unsigned char tensor_smem[];
  __shared__ TensorBarriers bar;
  __shared__ uint16_t s_cached[8][kLoadWarps];  // by stage: its keys that are cache rows
  __shared__ uint32_t s_tmem;
  __shared__ unsigned long long s_bad;  // nodes whose V held a non-finite element
  __shared__ float2 s_stats[kTile];
  unsigned char *smem = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(tensor_smem) + 1023) & ~(uintptr_t)1023);
  unsigned char *ring = smem + Shape::ring;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, split = blockIdx.x;
  const int D = p.head_dim, G = p.groups, all = p.nodes * G;
  const int tiles = (int)ceil_div(all, p.tile_rows);
  const int kh = blockIdx.y / tiles, r0 = blockIdx.y % tiles * p.tile_rows, b = blockIdx.z;
  const int n_nodes = nodes_of(p, b), live = n_nodes * G;
  const bool apart = p.tile_rows > kTile;  // the streams own different rows
  const int64_t valid = rows_of(p, b);
  const int64_t total = r0 < live ? valid + n_nodes : 0;
  const int64_t chunk = ceil_div(ceil_div(total, p.splits), kKeys) * kKeys;
  const int64_t begin = min(total, split * chunk), end = min(total, begin + chunk);
  const int blocks = (int)ceil_div(end - begin, kKeys);
  const int items = apart ? 2 * blocks : blocks;
  T *out = static_cast<T *>(p.out) + (int64_t)b * p.nodes * p.q_heads * D;
  auto out_row = [&](int row) {
    return out + (int64_t)(row / G) * p.q_heads * D + (int64_t)(kh * G + row % G) * D;
  };

  if (blocks == 0) {  // nothing is seen here: zeros, or a split without weight
    for (int i = warp; i < p.tile_rows && r0 + i < all; i += kTensorThreads / 32) {
      if (p.splits == 1)
        for (int d = lane; d < D; d += 32) out_row(r0 + i)[d] = from_f32<T>(0.f);
      else if (lane == 0)
        p.stats[partial_number(p, b, kh, r0 + i, split)] = make_float2(-INFINITY, 0.f);
    }
    return;
  }

  // live rows of each stream's tile; a warp without any only takes part in barriers
  const int live0 = min(kTile, live - r0);
  const int live1 = apart ? max(0, min(kTile, live - r0 - kTile)) : live0;
  if (warp == kSoftmaxWarps + kLoadWarps) {
    if (lane == 0) {
      for (int i = 0; i < Shape::stages; ++i) {
        mbar_init(&bar.kv_full[i], kLoadThreads);
        mbar_init(&bar.kv_free[i], apart ? 2 : 1);
      }
      for (int w = 0; w < 2; ++w) {
        const int threads = 32 * max(1, (int)ceil_div(w ? live1 : live0, 32));
        mbar_init(&bar.s_full[w], 1);
        mbar_init(&bar.s_free[w], threads);
        for (int i = 0; i < 2; ++i) {
          mbar_init(&bar.p_full[w][i], threads);
          mbar_init(&bar.pv_done[w][i], 1);
        }
      }
      s_bad = 0;
      asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     smem_addr(&s_tmem)),
                 "r"(2 * kStreamColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
  } else if (warp < kSoftmaxWarps) {
    // Q into both streams' tiles (one tile when they share it), dead rows zero
    const T *query = static_cast<const T *>(p.query) + b * p.q_batch_stride;
    constexpr int chunks = kDim / 8;
    for (int i = tid; i < p.tile_rows * chunks; i += 32 * kSoftmaxWarps) {
      const int r = i / chunks, c = i % chunks, row = r0 + r;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (row < live && c * 8 < D)
        x = *reinterpret_cast<const uint4 *>(query + row / G * p.q_node_stride +
                                             (int64_t)(kh * G + row % G) * D + c * 8);
      *reinterpret_cast<uint4 *>(smem + r / kTile * Shape::q_bytes + place(r % kTile, c, kTile)) =
          x;
    }
    fence_async_proxy();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;

  if (warp < kSoftmaxWarps) {
    // ---- softmax of stream w --------------------------------------------------------
    const int w = warp / 4, quarter = warp % 4;
    const int mine = apart ? blocks : (blocks + 1 - w) / 2;
    const int live_here = w ? live1 : live0;
    const int r = quarter * 32 + lane;           // row of the tile
    const int row = r0 + (apart ? w * kTile : 0) + r;
    const uint32_t lanes = tmem + w * kStreamColumns + ((uint32_t)(quarter * 32) << 16);
    const bool here = quarter < max(1, (int)ceil_div(live_here, 32));
    const uint64_t see =
        r < live_here ? (uint64_t)p.mask[(int64_t)b * p.nodes + row / G] : 0;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int k = 0; here && ok && k < mine; ++k) {
      const int block = apart ? k : 2 * k + w, slot = block % Shape::stages, buffer = k & 1;
      ok = mbar_wait(&bar.kv_full[slot], block / Shape::stages & 1, p.status) &&
           mbar_wait(&bar.s_full[w], k & 1, p.status);
      if (!__all_sync(kFullMask, ok)) break;
      // keys this row sees: cache rows, then nodes from position n0 on
      uint64_t seen = *reinterpret_cast<const uint64_t *>(s_cached[slot]);
      const int64_t k0 = begin + (int64_t)block * kKeys;
      if (k0 + kKeys > valid) {
        const int n0 = (int)(valid > k0 ? valid - k0 : 0), j0 = (int)(k0 + n0 - valid);
        const int n = (int)(min(end, k0 + kKeys) - (k0 + n0));  // nodes in the block
        const uint64_t nodes = n >= 64 ? ~0ull : (1ull << n) - 1;
        seen |= (see >> j0 & nodes) << n0;
      }
      uint32_t s[2][32];
      fence_after();
      tmem_load32(s[0], lanes + kColumnsS);
      tmem_load32(s[1], lanes + kColumnsS + 32);
      tmem_load_wait(s[0]);
      tmem_load_wait(s[1]);
      fence_before();
      mbar_arrive(&bar.s_free[w]);
      float top = -INFINITY;
      if (__all_sync(kFullMask, seen == ~0ull)) {
#pragma unroll
        for (int i = 0; i < 64; ++i) top = fmaxf(top, __uint_as_float(s[i / 32][i % 32]));
      } else {
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          if (!(seen >> i & 1)) s[i / 32][i % 32] = 0xff800000u;  // -inf
          top = fmaxf(top, __uint_as_float(s[i / 32][i % 32]));
        }
      }
      top *= p.scale_log2;
      if (__any_sync(kFullMask, top > m + kLazy)) {
        const float to = fmaxf(m, top);
        const float f = m == -INFINITY ? 0.f : tree_exp2(m - to);
        if (k > 0) {  // the output so far
          ok = mbar_wait(&bar.pv_done[w][buffer ^ 1], (k - 1) >> 1 & 1, p.status);
          if (!__all_sync(kFullMask, ok)) break;
          fence_after();
#pragma unroll
          for (int c = 0; c < kDim; c += 32) {
            uint32_t o[32];
            tmem_load32(o, lanes + c);
            tmem_load_wait(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_store32(lanes + c, o);
          }
          tmem_store_wait();
        }
        l *= f;
        m = to;
      }
      // a row that has seen nothing keeps m = -inf: its weights are exp2(-inf) = 0
      const float base = m == -INFINITY ? 0.f : kLift<T> - m;
      uint32_t packed[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float a = tree_exp2(fmaf(__uint_as_float(s[i / 16][2 * i % 32]), p.scale_log2, base));
        const float c =
            tree_exp2(fmaf(__uint_as_float(s[i / 16][2 * i % 32 + 1]), p.scale_log2, base));
        l += a + c;
        packed[i] = pack2<T>(a, c);
      }
      if (k >= 2) {  // the products that read this buffer last
        ok = mbar_wait(&bar.pv_done[w][buffer], (k - 2) >> 1 & 1, p.status);
        if (!__all_sync(kFullMask, ok)) break;
        fence_after();
      }
      tmem_store32(lanes + kColumnsP + buffer * 32, packed);
      tmem_store_wait();
      fence_before();
      mbar_arrive(&bar.p_full[w][buffer]);
    }
    // ---- the result ---------------------------------------------------------------------
    if (ok && mine > 0)
      ok = mbar_wait(&bar.pv_done[w][(mine - 1) & 1], (mine - 1) >> 1 & 1, p.status);
    __syncwarp();
    fence_after();
    // Streams of the same rows join through the ring's memory: its last products
    // are done when both streams' are, which the named barrier brings together.
    float *join = reinterpret_cast<float *>(ring);
    asm volatile("bar.sync 1, %0;\n" ::"n"(32 * kSoftmaxWarps) : "memory");
    if (!apart) {
      if (w == 1 && here) {
        s_stats[r] = make_float2(m, l);
#pragma unroll
        for (int c = 0; c < kDim; c += 32) {
          uint32_t o[32];
          tmem_load32(o, lanes + c);
          tmem_load_wait(o);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            join[r * Shape::join_pitch + c + i] = mine > 0 ? __uint_as_float(o[i]) : 0.f;
        }
      }
      __syncwarp();
      asm volatile("bar.sync 1, %0;\n" ::"n"(32 * kSoftmaxWarps) : "memory");
    }
    if (here && (apart || w == 0)) {
      float f = 1.f, g = 0.f;
      if (!apart) {
        const float2 other = s_stats[r];
        const float to = fmaxf(m, other.x);
        f = m == -INFINITY ? 0.f : tree_exp2(m - to);
        g = other.x == -INFINITY ? 0.f : tree_exp2(other.x - to);
        // a sum of NaN scores has no maximum: let it through
        l = (m == -INFINITY ? l : l * f) + (other.x == -INFINITY ? other.y : other.y * g);
        m = to;
      }
      const bool in = row < all;
      const uint64_t bad = r < live_here ? s_bad & see : 0;
      const float inv = r < live_here && (l > 0.f || l != l) ? 1.f / l : 0.f;
      const int64_t at = in ? partial_number(p, b, kh, row, split) : 0;
#pragma unroll
      for (int c = 0; c < kDim; c += 32) {
        uint32_t o[32];
        __syncwarp();
        tmem_load32(o, lanes + c);
        tmem_load_wait(o);
        if (!in || c >= D) continue;
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          x[i] = __uint_as_float(o[i]) * f;
          if (!apart) x[i] = fmaf(g, join[r * Shape::join_pitch + c + i], x[i]);
        }
        if (r >= live_here)
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = 0.f;
        if (p.splits == 1) {
          T *to = out_row(row) + c;
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            if (c + i < D) {
              uint4 v;
              v.x = pack2<T>(x[i] * inv, x[i + 1] * inv);
              v.y = pack2<T>(x[i + 2] * inv, x[i + 3] * inv);
              v.z = pack2<T>(x[i + 4] * inv, x[i + 5] * inv);
              v.w = pack2<T>(x[i + 6] * inv, x[i + 7] * inv);
              *reinterpret_cast<uint4 *>(to + i) = v;
            }
        } else {
          float *to = p.partials + at * D + c;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            if (c + i < D)
              *reinterpret_cast<float4 *>(to + i) =
                  make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        }
      }
      if (bad != 0)
        for (int d = 0; d < D; ++d) {
          const float x = nonfinite_sum<T>(p, b, kh, d, bad);
          if (p.splits == 1) out_row(row)[d] = from_f32<T>(to_f32(out_row(row)[d]) + x);
          else p.partials[at * D + d] += x;
        }
      if (in && p.splits > 1) p.stats[at] = make_float2(m, r < live_here ? l : 0.f);
    }
    // rows of padded nodes that no live warp covers
    if (!here && (apart || w == 0) && row < all) {
      if (p.splits == 1)
        for (int d = 0; d < D; d += 8)
          *reinterpret_cast<uint4 *>(out_row(row) + d) = make_uint4(0, 0, 0, 0);
      else
        p.stats[partial_number(p, b, kh, row, split)] = make_float2(-INFINITY, 0.f);
    }
  } else if (warp < kSoftmaxWarps + kLoadWarps) {
    // ---- key blocks into the ring ---------------------------------------------------
    const int lw = warp - kSoftmaxWarps;
    constexpr int chunks = kDim / 8, together = 32 / chunks;  // keys of a warp's copy
    const int c = lane % chunks;
    const bool in_dim = c * 8 < D;
    const int64_t row_elems = (int64_t)p.kv_heads * D, plane = p.page_size * row_elems;
    const T *pool = static_cast<const T *>(p.pool) + (int64_t)kh * D + c * 8;
    const int64_t node_base = (int64_t)b * p.kv_batch_stride + (int64_t)kh * D + c * 8;
    const T *key = static_cast<const T *>(p.key) + node_base;
    const T *value = static_cast<const T *>(p.value) + node_base;
    const int64_t *rows = p.rows + b * p.rows_batch_stride;
    constexpr int mine = kKeys / kLoadWarps;  // keys of a block that this warp copies
    // lane i < mine reads the row number of the warp's i-th key, a block ahead
    auto look = [&](int block) -> int64_t {
      const int64_t at = begin + (int64_t)block * kKeys + lw * mine + lane;
      return lane < mine && at < end && at < valid ? __ldg(rows + at) : -1;
    };
    int64_t next = look(0);
    int announced = 0;
    bool ok = true;
    for (int block = 0; block < blocks; ++block) {
      const int slot = block % Shape::stages;
      if (block >= Shape::stages) {
        ok = mbar_wait(&bar.kv_free[slot], (block / Shape::stages - 1) & 1, p.status);
        if (!__all_sync(kFullMask, ok)) break;
      }
      const int64_t offset = row_offset(p, next, row_elems);
      next = look(block + 1);
      const unsigned cached = __ballot_sync(kFullMask, offset >= 0);
      if (lane == 0) s_cached[slot][lw] = (uint16_t)cached;
      unsigned char *stage = ring + slot * 2 * Shape::plane_bytes;
      const int64_t at0 = begin + (int64_t)block * kKeys + lw * mine;
#pragma unroll
      for (int i = 0; i < mine; i += together) {
        const int mk = i + lane / chunks, k = lw * mine + mk;
        const int64_t off = __shfl_sync(kFullMask, offset, mk);
        const uint32_t to = place(k, c, kKeys);
        if (at0 + mk >= valid && at0 + mk < end) {  // a node
          const int64_t j = at0 + mk - valid;
          uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
          if (in_dim) {
            kx = *reinterpret_cast<const uint4 *>(key + j * p.kv_node_stride);
            vx = *reinterpret_cast<const uint4 *>(value + j * p.kv_node_stride);
          }
          if (clear_nonfinite<T>(vx)) atomicOr(&s_bad, 1ull << j);
          *reinterpret_cast<uint4 *>(stage + to) = kx;
          *reinterpret_cast<uint4 *>(stage + Shape::plane_bytes + to) = vx;
        } else {
          const bool in = off >= 0;
          const T *src = in ? pool + off : pool;
          tree_cp_async16(smem_addr(stage + to), src, in && in_dim);
          tree_cp_async16(smem_addr(stage + Shape::plane_bytes + to), in ? src + plane : src,
                          in && in_dim);
        }
      }
      asm volatile("cp.async.commit_group;\n" ::: "memory");
      if (block >= Shape::ahead) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(Shape::ahead) : "memory");
        fence_async_proxy();
        mbar_arrive(&bar.kv_full[announced % Shape::stages]);
        ++announced;
      }
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    fence_async_proxy();
    if (ok)
      for (; announced < blocks; ++announced) mbar_arrive(&bar.kv_full[announced % Shape::stages]);
  } else if (lane == 0) {
    // ---- the products ---------------------------------------------------------------
    const uint32_t i_scores = instruction<T>(kKeys, false), i_output = instruction<T>(kDim, true);
    const uint32_t q_base = smem_addr(smem), kv_base = smem_addr(ring);
    auto scores = [&](int n) -> bool {
      const int w = n & 1, k = n >> 1, block = apart ? k : n, slot = block % Shape::stages;
      if (!mbar_wait(&bar.kv_full[slot], block / Shape::stages & 1, p.status)) return false;
      if (k > 0 && !mbar_wait(&bar.s_free[w], (k - 1) & 1, p.status)) return false;
      fence_after();
      const uint32_t q = q_base + (apart ? w * Shape::q_bytes : 0);
      const uint32_t kp = kv_base + slot * 2 * Shape::plane_bytes;
#pragma unroll
      for (int kk = 0; kk < kDim / 16; ++kk)
        mma_shared(tmem + w * kStreamColumns + kColumnsS,
                   descriptor(q + kk / 4 * kTile * 128 + kk % 4 * 32, 16, 1024),
                   descriptor(kp + kk / 4 * kKeys * 128 + kk % 4 * 32, 16, 1024), i_scores,
                   kk > 0);
      commit(&bar.s_full[w]);
      return true;
    };
    auto output = [&](int n) -> bool {
      const int w = n & 1, k = n >> 1, block = apart ? k : n, slot = block % Shape::stages;
      if (!mbar_wait(&bar.p_full[w][k & 1], k >> 1 & 1, p.status)) return false;
      fence_after();
      const uint32_t vp = kv_base + slot * 2 * Shape::plane_bytes + Shape::plane_bytes;
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk)
        mma_tmem(tmem + w * kStreamColumns,
                 tmem + w * kStreamColumns + kColumnsP + (k & 1) * 32 + kk * 8,
                 descriptor(vp + kk * 2048, kKeys * 128, 1024), i_output, k > 0 || kk > 0);
      commit(&bar.pv_done[w][k & 1]);
      commit(&bar.kv_free[slot]);
      return true;
    };
    bool ok = true;
    for (int n = 0; ok && n < 2 && n < items; ++n) ok = scores(n);
    for (int n = 0; ok && n < items; ++n) {
      if (n + 2 < items) ok = scores(n + 2);
      if (ok) ok = output(n);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == kSoftmaxWarps + kLoadWarps) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem),
                 "r"(2 * kStreamColumns));
  }
}

template <typename T, int kDim> int launch(const TreeParams &p, cudaStream_t s) {
  auto kernel = tree_tensor_kernel<T, kDim>;
  const size_t bytes = TensorShape<kDim>::dynamic;
  if (int e = reserve_smem(reinterpret_cast<const void *>(kernel), bytes, "attend_tree")) return e;
  const int64_t tiles = ceil_div((int64_t)p.nodes * p.groups, p.tile_rows);
  const dim3 grid((unsigned)p.splits, (unsigned)(p.kv_heads * tiles), (unsigned)p.batch);
  kernel<<<grid, kTensorThreads, bytes, s>>>(p);
  return check_launch("tree_tensor_kernel");
}

}  // namespace

int launch_tree_tensor(const TreeParams &p, int dtype, cudaStream_t s) {
  if (dtype == HS_FLOAT16)
    return p.head_dim <= 64 ? launch<__half, 64>(p, s) : launch<__half, 128>(p, s);
  return p.head_dim <= 64 ? launch<__nv_bfloat16, 64>(p, s) : launch<__nv_bfloat16, 128>(p, s);
}

}  // namespace hs
