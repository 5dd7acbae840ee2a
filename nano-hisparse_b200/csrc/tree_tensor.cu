// Tree attention on the fifth-generation tensor cores: 16-bit types, head_dim a multiple
// of 8 up to 256.
//
// A block serves 128 query rows (the M = 128 tile of tcgen05.mma, its rows the TMEM
// lanes) of a request and KV head over a split of the key list, in blocks of 64 keys.
// Up to head_dim 128 two blocks share an SM, so that one's softmax runs beside the
// other's products, and one's start and end beside the other's middle. 10 warps:
//   warps 0-3       softmax: a thread has one query row. Scores from TMEM, P =
//                   exp2(s - m) rounded to the 16-bit type (half a step of each weight,
//                   as large as the rounding of the result) back to TMEM. The maximum is
//                   raised only when a score passes it by more than 8 (a factor of 256,
//                   inside fp16's range), so the output, which stays in TMEM, is rescaled
//                   rarely.
//   warps 4-7       copy key blocks (two warps K, two V) into rings of stages in the
//                   128-byte-swizzled layout of the descriptors: 16 rows that follow one
//                   another in the pool with one tiled copy, others with cp.async, 16
//                   bytes a thread. (The copy engine's gather of four rows of 128 bytes
//                   was measured at 73 clocks each, a third of this rate.)
//   warp 8          issues S = Q K^T, both operands in shared memory, K-major
//   warp 9          issues O += P V, P in TMEM, V in shared memory, MN-major (as
//                   stored: a key's elements are adjacent)
// A block's scores do not wait for the one before it, so the tensor pipe and the
// softmax overlap. What bounds it: up to about 50 nodes the reads of K and V, beyond
// that the chain score, softmax, product (special functions 41 %, tensor pipe 60 %);
// with few keys the chain of its start (counts, row numbers, keys: 4 us).
// 8 requests of 32 nodes, 32,768 rows, 32 query and 8 KV heads of 128 in bf16: 182 us with
// the join, 5.3 TB/s (6.7 in the steady part); 213 with one block of two tiles on an SM,
// 217 with pages of 8 rows, whose copies all go through cp.async, where pages of 16 take
// 203 (every node and row present). 8 requests of 63 nodes, 8,192 rows, 28 query and 4 KV
// heads: 78 us, 757 TFLOP/s. 8 requests of 8 nodes, 8,192 rows, 16 query and 4 KV heads of
// 256: 67 us, 4.0 TB/s.
//
// TMEM columns: O first, then two buffers of S; P takes the second half of its S.
// Every wait is bounded; one that runs out sets HS_DEV_WAIT_TIMEOUT, ends its
// warp's loop, and so lets every other wait run out.
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "tree.cuh"

namespace hs {
namespace {

constexpr int kSoftmaxWarps = 4, kLoadWarps = 4;  // half of the latter for K, half for V
constexpr int kMaxStages = 5;
constexpr int kPanel = 1024;   // bytes of 8 rows x 64 elements
constexpr int kRun = 16;       // rows of a tiled copy
constexpr int kMarks = 16;     // blocks whose marks (which keys are cache rows) are kept
constexpr int kScoreWarp = kSoftmaxWarps + kLoadWarps, kOutputWarp = kScoreWarp + 1;
constexpr int kTensorThreads = 32 * (kOutputWarp + 1);
constexpr int kTile = 128;     // query rows
constexpr int kKeys = 64;      // keys of a block
constexpr int kLook = 6;       // blocks that row numbers are read ahead
constexpr unsigned long long kWaitNanoseconds = 4000000000ull;  // then a wait gives up

struct TensorShared {
  uint64_t k_full[kMaxStages], k_free[kMaxStages], v_full[kMaxStages], v_free[kMaxStages];
  uint64_t s_full[2], p_full[2], pv_done[2];  // by buffer
  unsigned long long bad;                     // nodes whose V held a non-finite element
  uint32_t cached[kMarks][kLoadWarps / 2];    // by block: its keys that are cache rows
  uint32_t tmem;
};

// Shared memory and TMEM of a block. kDim: head_dim rounded up to 64, 128 or 256, the rest
// zero. An operand is a list of 8-row groups, each of kDim / 64 panels of 64 elements
// (128 bytes) a row: a panel of a group is a swizzle atom, and a run of rows in the
// pool lands in it with one tiled copy.
// K and V have rings of their own: a stage of K is free when its scores are done, a
// stage of V only when its output is.
template <int kDim> struct TensorShape {
  static constexpr int atom = kDim / 64 * kPanel;        // bytes of an 8-row group
  static constexpr int q_bytes = kTile * kDim * 2;
  static constexpr int plane_bytes = kKeys * kDim * 2;   // a stage: K or V of a block
  static constexpr int resident = kDim <= 128 ? 2 : 1;   // blocks on an SM
  static constexpr int k_stages = kDim == 64 ? 4 : 2;
  static constexpr int v_stages = kDim == 64 ? 5 : kDim == 128 ? 3 : 2;
  static constexpr int column_s = kDim <= 128 ? 128 : 256;  // O before it
  static constexpr int columns = 2 * column_s;
  static constexpr int bytes = q_bytes + (k_stages + v_stages) * plane_bytes;
  static constexpr size_t dynamic = bytes + 1024;        // and TensorShared
  static_assert(k_stages <= kMaxStages && v_stages <= kMaxStages, "barriers");
  static_assert(sizeof(TensorShared) <= 1024, "TensorShared has its place");
  static_assert(resident * (dynamic + 1024) <= 228 * 1024 && resident * columns <= 512,
                "the blocks fit an SM");
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
__device__ __forceinline__ void tmem_load16(uint32_t (&r)[16], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, "
               "%9, %10, %11, %12, %13, %14, %15}, [%16];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, "
               "%8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
               ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
                 "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15])
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
__device__ __forceinline__ void tmem_load16_done(uint32_t (&a)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]),
                 "+r"(a[6]), "+r"(a[7]), "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]),
                 "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15])
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
// Scores of keys that are not seen become -inf.
__device__ __forceinline__ void hide(uint32_t (&s)[32], uint32_t seen) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!(seen >> i & 1)) s[i] = 0xff800000u;
}
__device__ __forceinline__ float largest(uint32_t (&s)[32], bool plain, uint32_t seen) {
  if (!plain) hide(s, seen);
  float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 32; i += 2)
    tops[i / 2 % 4] = max3(tops[i / 2 % 4], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
  return fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
}

// As mbar_wait, without the hint to sleep: waits here are a few hundred clocks, and
// waking from a hinted sleep was measured to take more than a thousand.
__device__ __forceinline__ bool wait_phase(uint64_t *bar, unsigned parity, int32_t *status) {
  unsigned long long first = 0;
  for (unsigned i = 0;; ++i) {
    unsigned done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 1023) == 1023) {
      unsigned long long now;
      asm volatile("mov.u64 %0, %%globaltimer;\n" : "=l"(now));
      if (first == 0) first = now;
      if (now - first > kWaitNanoseconds) break;
    }
  }
  flag(status, HS_DEV_WAIT_TIMEOUT);
  return false;
}
__device__ __forceinline__ void mbar_arrive_many(uint64_t *bar, unsigned count) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_addr(bar)), "r"(count)
               : "memory");
}
// kRun rows of one KV head (panels `panel` on) from row 8 * group of the pool's rows,
// completing on `bar`
__device__ __forceinline__ void tile_copy(uint32_t dst, const CUtensorMap *map, int panel,
                                          int group, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%2, %2, %3, %4}], [%5];\n" ::"r"(dst),
      "l"(map), "r"(0), "r"(panel), "r"(group), "r"(smem_addr(bar))
      : "memory");
}
// Arrives on `bar` once this thread's copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_addr(bar))
               : "memory");
}
// Arrives on `bar` once the products issued so far are done.
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(
                   smem_addr(bar))
               : "memory");
}
// Shared-memory descriptor, 128-byte swizzle: the low word has the address and, for
// MN-major operands that span several panels, the panels' distance; the high word
// the distance of 8-row groups. Adding bytes / 16 to the low word moves the address.
template <int kDim>
constexpr uint32_t kDescriptorHigh = (TensorShape<kDim>::atom >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t descriptor(uint32_t addr) {
  return (addr >> 4) | (kPanel >> 4) << 16;
}
// D = A B (+ D), both operands in shared memory
template <int kDim>
__device__ __forceinline__ void mma_shared(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                           bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n"
      " mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescriptorHigh<kDim>)
      : "memory");
}
// A in TMEM
template <int kDim>
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                         bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %4, 0;\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescriptorHigh<kDim>)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(chosen));
  return chosen != 0;
}
// Instruction descriptor: fp32 accumulator, M = 128, n columns; b_mn: B is MN-major
template <typename T> __device__ __forceinline__ uint32_t instruction(int n, bool b_mn) {
  constexpr uint32_t type = std::is_same<T, __half>::value ? 0 : 1;  // fp16, bf16
  return 1u << 4 | type << 7 | type << 10 | (uint32_t)b_mn << 16 | (uint32_t)(n >> 3) << 17 |
         (uint32_t)(kTile >> 4) << 24;
}
// Place of 16-byte chunk c of row r of an operand
template <int kDim> __device__ __forceinline__ uint32_t place(int r, int c) {
  return (uint32_t)((r >> 3) * TensorShape<kDim>::atom + (c >> 3) * kPanel + (r & 7) * 128 +
                    (((c & 7) ^ (r & 7)) << 4));
}

// This thread's 16-byte chunks of the 128 rows from row r0 of Q into a tile,
// kThreads threads taking part; rows past the last live one become zero. One division:
// from row to row the pointer moves by a constant, but for a node's last head.
template <typename T, int kDim, int kThreads>
__device__ __forceinline__ void copy_q(const TreeParams &p, int b, int kh, int r0, int live,
                                       unsigned char *tile, int thread) {
  constexpr int chunks = kDim / 8, step = kThreads / chunks;
  static_assert(step % 4 == 0, "a thread's rows have one or two places in the swizzle");
  const int D = p.head_dim, G = p.groups, c = thread % chunks, r = thread / chunks;
  int left = c * 8 < D ? live - (r0 + r) : 0;  // rows to the last live one
  const int t = (r0 + r) / G, skip = step / G;
  int g = r0 + r - t * G;
  const T *from = static_cast<const T *>(p.query) + b * p.q_batch_stride +
                  t * p.q_node_stride + (int64_t)(kh * G + g) * D + c * 8;
  const int64_t stride = skip * p.q_node_stride + (int64_t)(step - skip * G) * D;
  const int64_t wrap = p.q_node_stride - (int64_t)G * D;
  const int rest = step - skip * G;
  const uint32_t even = smem_addr(tile) + place<kDim>(r, c);
  const uint32_t odd = smem_addr(tile) + place<kDim>(r + step, c);
#pragma unroll
  for (int i = 0; i < kTile / step; ++i) {
    // two steps are whole groups of 8 rows
    const uint32_t to = (i % 2 ? odd : even) + i / 2 * (2 * step / 8) * TensorShape<kDim>::atom;
    tree_cp_async16(to, left > 0 ? from : static_cast<const T *>(p.query), left > 0);
    left -= step;
    from += stride;
    g += rest;
    if (g >= G) {
      g -= G;
      from += wrap;
    }
  }
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kTensorThreads, TensorShape<kDim>::resident)
    tree_tensor_kernel(TreeParams p, const __grid_constant__ CUtensorMap map, bool tiled) {
  using Shape = TensorShape<kDim>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *k_ring = smem + Shape::q_bytes;
  unsigned char *v_ring = k_ring + Shape::k_stages * Shape::plane_bytes;
  TensorShared &sh = *reinterpret_cast<TensorShared *>(smem + Shape::bytes);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, split = blockIdx.y;
  const int warp = __shfl_sync(kFullMask, tid >> 5, 0);  // the same for every lane, to the compiler too
  const int D = p.head_dim, G = p.groups, all = p.nodes * G, b = blockIdx.z;
  const int n_nodes = nodes_of(p, b), valid = (int)rows_of(p, b), live = n_nodes * G;
  const int tiles = (all + kTile - 1) / kTile;
  const int kh = blockIdx.x / tiles, r0 = blockIdx.x % tiles * kTile;
  // the keys of this split: begin .. end - 1
  const unsigned total = r0 < live ? (unsigned)(valid + n_nodes) : 0;
  const unsigned share = ((total + p.splits - 1) / p.splits + kKeys - 1) / kKeys * kKeys;
  const int begin = (int)min((unsigned long long)total, (unsigned long long)split * share);
  const int end = (int)min(total, begin + share);
  const int blocks = (end - begin + kKeys - 1) / kKeys;

  const bool placed = (smem_addr(smem) & 1023) == 0;  // the swizzle counts on it
  if (!placed && tid == 0) flag(p.status, HS_DEV_MISALIGNED);
  if (blocks == 0 || !placed) {  // nothing is seen here: zeros, or a split without weight
    for (int i = warp; i < kTile && r0 + i < all; i += kTensorThreads / 32) {
      if (p.splits > 1) {
        if (lane == 0)
          *stat_of(p, part_of(p, b, kh, split), r0 + i) = make_float2(-INFINITY, 0.f);
      } else {
        T *out = static_cast<T *>(p.out) + out_offset(p, b, kh, r0 + i);
        for (int d = lane; d < D; d += 32) out[d] = from_f32<T>(0.f);
      }
    }
    return;
  }

  // A softmax warp without a live row takes no part in the blocks.
  const int live_here = min(kTile, live - r0), live_warps = (live_here + 31) / 32;
  if (tid == 32 * kSoftmaxWarps)
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map) : "memory");
  if (tid == 32 * kScoreWarp) {
    for (int i = 0; i < kMaxStages; ++i) {
      mbar_init(&sh.k_full[i], kLoadWarps / 2 * (32 + 1));
      mbar_init(&sh.v_full[i], kLoadWarps / 2 * (32 + 1));
      mbar_init(&sh.k_free[i], 1);
      mbar_init(&sh.v_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 2);  // the products, and the marks that came with their keys
      mbar_init(&sh.p_full[i], live_warps);
      mbar_init(&sh.pv_done[i], 2);  // the products, and the marks that came with their values
    }
    sh.bad = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();

  if (warp >= kSoftmaxWarps && warp < kSoftmaxWarps + kLoadWarps) {
    // ---- K or V of the key blocks into its ring -------------------------------------
    constexpr int warps = kLoadWarps / 2;
    constexpr int chunks = kDim / 8, together = 32 / chunks, steps = kRun / together;
    static_assert(kKeys / warps == 32, "a lane for each key that a warp copies");
    const bool values = warp >= kSoftmaxWarps + warps;
    const int lw = (warp - kSoftmaxWarps) % warps, c = lane % chunks;
    const bool in_dim = c * 8 < D;
    const int64_t row_elems = (int64_t)p.kv_heads * D;
    const T *pool = static_cast<const T *>(p.pool) + (int64_t)kh * D + c * 8 +
                    (values ? p.page_size * row_elems : 0);
    const T *drafted = static_cast<const T *>(values ? p.value : p.key) +
                       (int64_t)b * p.kv_batch_stride + (int64_t)kh * D + c * 8;
    const int64_t *rows = p.rows + b * p.rows_batch_stride;
    uint64_t *full = values ? sh.v_full : sh.k_full, *free = values ? sh.v_free : sh.k_free;
    const int stages = values ? Shape::v_stages : Shape::k_stages;
    unsigned char *ring = values ? v_ring : k_ring;
    const uint32_t ring_addr = smem_addr(ring);
    // a lane reads the row number of one key of the warp's 32, kLook blocks ahead: a
    // block's time is shorter than the read's
    const int last = min(end, valid);
    auto look = [&](int block) -> int64_t {
      const int at = begin + block * kKeys + lw * 32 + lane;
      return at < last ? __ldg(rows + at) : -1;
    };
    int64_t next[kLook];
#pragma unroll
    for (int i = 0; i < kLook; ++i) next[i] = i < blocks ? look(i) : -1;
    // Where this lane's first chunk goes; i keys further it is i rows down, and the
    // row's part of the swizzle differs by i (the lane's own part is below `together`).
    const uint32_t to0 = place<kDim>(lw * 32 + lane / chunks, c);
    int slot = 0, turn = 1;
    for (int block = 0; block < blocks; ++block) {
      if (block >= stages) {
        const bool ok = wait_phase(&free[slot], turn, p.status);
        if (!__all_sync(kFullMask, ok)) {  // leave no copy behind
          for (int i = max(0, block - stages); i < block; ++i)
            wait_phase(&full[i % stages], i / stages & 1, p.status);
          break;
        }
      }
      const int64_t row = next[0], offset = row_offset(p, row, row_elems);
#pragma unroll
      for (int i = 0; i + 1 < kLook; ++i) next[i] = next[i + 1];
      next[kLook - 1] = block + kLook < blocks ? look(block + kLook) : -1;
      if (!values) {
        const unsigned cached = __ballot_sync(kFullMask, offset >= 0);
        if (lane == 0) sh.cached[block % kMarks][lw] = cached;
      }
      const uint32_t stage_addr = ring_addr + slot * Shape::plane_bytes;
      // Either half of the warp's rows: rows that follow one another from a multiple of 8
      // on, as those of a page do, take one tiled copy. The copy engine keeps more reads
      // in flight than cp.async does.
      const int64_t row0 = __shfl_sync(kFullMask, row, lane & 16);
      const bool run = tiled && (row0 & 7) == 0 &&
                       (row0 & (p.page_size - 1)) + kRun <= p.page_size && offset >= 0 &&
                       row == row0 + (lane & 15);
      const unsigned runs = __ballot_sync(kFullMask, run);
      const bool first_run = (runs & 0xffff) == 0xffff, second_run = runs >> 16 == 0xffff;
      if (first_run || second_run) {
        const int64_t row1 = __shfl_sync(kFullMask, row, 16);
        if (lane == 0) {
          mbar_add_tx(&full[slot], ((int)first_run + (int)second_run) * kRun * kDim * 2);
          const auto copy = [&](int64_t from, int half) {
            const int group = (int)(((from >> p.page_shift) * 2 * p.page_size +
                                     (values ? p.page_size : 0) + (from & (p.page_size - 1))) >> 3);
            tile_copy(stage_addr + (lw * 32 + half * kRun) * kDim * 2, &map, kh * (kDim / 64),
                      group, &full[slot]);
          };
          if (first_run) copy(row0, 0);
          if (second_run) copy(row1, 1);
          if (first_run && second_run) mbar_arrive_many(&full[slot], 32 + 1);
        }
      }
      if (!first_run || !second_run) {
        bool written = false;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (half == 0 ? first_run : second_run) continue;
          const int first = begin + block * kKeys + lw * 32 + half * kRun;  // its first key
          if (first + kRun <= valid) {
#pragma unroll
            for (int i = 0; i < steps; ++i) {
              const int key = i * together;
              const int64_t off = __shfl_sync(kFullMask, offset, half * kRun + key + lane / chunks);
              tree_cp_async16(stage_addr + half * (kRun / 8 * Shape::atom) +
                                  (to0 ^ ((key & 7) << 4)) + (key >> 3) * Shape::atom +
                                  (key & 7) * 128,
                              off >= 0 ? pool + off : pool, off >= 0 && in_dim);
            }
          } else {
            written = true;
            constexpr int some = steps < 4 ? steps : 4;  // loads in flight
#pragma unroll 1
            for (int i0 = 0; i0 < steps; i0 += some) {
              const auto key = [&](int i) { return (i0 + i) * together + lane / chunks; };
              const auto node = [&](int i) {  // this lane's key as a node, or -1
                const int at = first + key(i);
                return at >= valid && at < end ? at - valid : -1;
              };
              uint4 raw[some];
#pragma unroll
              for (int i = 0; i < some; ++i) {
                raw[i] = make_uint4(0, 0, 0, 0);
                if (node(i) >= 0 && in_dim)
                  raw[i] = *reinterpret_cast<const uint4 *>(drafted + node(i) * p.kv_node_stride);
              }
#pragma unroll
              for (int i = 0; i < some; ++i) {
                const uint32_t to = place<kDim>(lw * 32 + half * kRun + key(i), c);
                const int64_t off = __shfl_sync(kFullMask, offset, half * kRun + key(i));
                if (node(i) >= 0) {
                  if (values && clear_nonfinite<T>(raw[i])) atomicOr(&sh.bad, 1ull << node(i));
                  *reinterpret_cast<uint4 *>(ring + slot * Shape::plane_bytes + to) = raw[i];
                } else {
                  tree_cp_async16(stage_addr + to, off >= 0 ? pool + off : pool,
                                  off >= 0 && in_dim);
                }
              }
            }
          }
        }
        // Every lane's copies announce themselves when they land; lane 0's arrival
        // carries what was written with plain stores.
        if (written) fence_async_proxy();
        __syncwarp();
        copies_arrive(&full[slot]);
        if (lane == 0) mbar_arrive(&full[slot]);
      }
      __syncwarp();
      if (++slot == stages) {
        slot = 0;
        turn ^= 1;
      }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    return;
  }

  if (warp < kSoftmaxWarps) {
    copy_q<T, kDim, kTile>(p, b, kh, r0, live, smem, tid);
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    fence_async_proxy();
  } else if (warp == kOutputWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     smem_addr(&sh.tmem)),
                 "r"(Shape::columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
  }
  fence_before();
  __syncwarp();
  asm volatile("bar.sync 2, %0;\n" ::"n"(32 * (kSoftmaxWarps + 2)) : "memory");
  fence_after();
  const uint32_t tmem = __shfl_sync(kFullMask, sh.tmem, 0);

  if (warp < kSoftmaxWarps) {
    // ---- softmax --------------------------------------------------------------------
    const int r = tid, row = r0 + r;  // this thread's row, of the tile and of all
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const bool here = warp < live_warps, alive = r < live_here;
    const uint64_t see = alive ? (uint64_t)p.mask[(int64_t)b * p.nodes + row / G] : 0;
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int k = 0; here && k < blocks; ++k) {
      const int buffer = k & 1;
      const uint32_t scores = lanes + Shape::column_s + buffer * kKeys, weights = scores + kKeys / 2;
      ok = wait_phase(&sh.s_full[buffer], k >> 1 & 1, p.status);
      if (!__all_sync(kFullMask, ok)) break;
      fence_after();
      uint32_t s[32];
      tmem_load32(s, scores);
      // keys this row sees: cache rows, then nodes from position n0 on
      const uint2 cached = *reinterpret_cast<const uint2 *>(sh.cached[k % kMarks]);
      uint64_t seen = (uint64_t)cached.y << 32 | cached.x;
      const int k0 = begin + k * kKeys;
      if (k0 + kKeys > valid) {
        const int n0 = max(valid - k0, 0), j0 = k0 + n0 - valid;
        const int n = min(end, k0 + kKeys) - (k0 + n0);  // nodes in the block
        const uint64_t nodes = n >= 64 ? ~0ull : (1ull << n) - 1;
        seen |= (see >> j0 & nodes) << n0;
      }
      const bool plain = __all_sync(kFullMask, seen == ~0ull);
      tmem_load_wait(s);
      float top = largest(s, plain, (uint32_t)seen);
      tmem_load32(s, scores + 32);
      tmem_load_wait(s);
      top = fmaxf(top, largest(s, plain, (uint32_t)(seen >> 32))) * p.scale_log2;
      if (__any_sync(kFullMask, top > m + kLazy)) {
        const float to = fmaxf(m, top);
        const float f = m == -INFINITY ? 0.f : tree_exp2(m - to);
        if (k > 0) {  // the output so far
          ok = wait_phase(&sh.pv_done[buffer ^ 1], (k - 1) >> 1 & 1, p.status);
          if (!__all_sync(kFullMask, ok)) break;
          fence_after();
#pragma unroll 1
          for (int c = 0; c < kDim; c += 16) {
            uint32_t o[16];
            tmem_load16(o, lanes + c);
            tmem_load16_done(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_store16(lanes + c, o);
          }
        }
        l *= f;
        m = to;
      }
      // a row that has seen nothing keeps m = -inf: its weights are exp2(-inf) = 0
      const float base = m == -INFINITY ? 0.f : kLift<T> - m;
      // P takes the columns of the second half of S, which is in registers; the
      // first half is read again (64 scores at once cost too many registers)
#pragma unroll
      for (int h = 1; h >= 0; --h) {
        if (h == 0) {
          tmem_load32(s, scores);
          tmem_load_wait(s);
          if (!plain) hide(s, (uint32_t)seen);
        }
        float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 e =
              pack_fma(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])),
                       scale2, make_float2(base, base));
          const float2 w2 = make_float2(tree_exp2(e.x), tree_exp2(e.y));
          sums[i % 2] = pack_add(sums[i % 2], w2);
          packed[i] = pack2<T>(w2.x, w2.y);
        }
        tmem_store16(weights + h * 16, packed);
        sums[0] = pack_add(sums[0], sums[1]);
        l += sums[0].x + sums[0].y;
      }
      tmem_store_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[buffer]);
    }
    // ---- the result -----------------------------------------------------------------
    if (ok) wait_phase(&sh.pv_done[(blocks - 1) & 1], (blocks - 1) >> 1 & 1, p.status);
    __syncwarp();
    fence_after();
    if (!alive) l = 0.f;
    const uint64_t bad = alive ? sh.bad & see : 0;
    if (p.splits > 1) {  // the unnormalised output; rows past the last live one have none
      const int64_t part = part_of(p, b, kh, split);
      if (here) {
        float4 *to = quad_of(p, part, row, 0);
#pragma unroll 1
        for (int c = 0; c < kDim; c += 32, to += 8 * all) {
          uint32_t x[32];
          tmem_load32(x, lanes + c);
          tmem_load_wait(x);
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            if (alive && c + i < D)
              to[i / 4 * all] = make_float4(__uint_as_float(x[i]), __uint_as_float(x[i + 1]),
                                            __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
        }
      }
      if (row < all) *stat_of(p, part, row) = make_float2(alive ? m : -INFINITY, l);
      if (bad != 0)
        for (int d = 0; d < D; ++d)
          reinterpret_cast<float *>(quad_of(p, part, row, d / 4))[d % 4] +=
              nonfinite_sum<T>(p, b, kh, d, bad);
    } else if (row - lane < all) {  // the result, zeros past the last live row
      T *out = static_cast<T *>(p.out) + out_offset(p, b, kh, min(row, all - 1));
      const float scale = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < kDim; c += 32) {
        uint32_t x[32];
        if (here) {
          tmem_load32(x, lanes + c);
          tmem_load_wait(x);
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          uint4 y = make_uint4(0, 0, 0, 0);
          if (alive) {
            const auto two = [&](int j) {
              return pack2<T>(__uint_as_float(x[i + j]) * scale, __uint_as_float(x[i + j + 1]) * scale);
            };
            y = make_uint4(two(0), two(2), two(4), two(6));
          }
          if (row < all && c + i < D) *reinterpret_cast<uint4 *>(out + c + i) = y;
        }
      }
      if (bad != 0)
        for (int d = 0; d < D; ++d)
          out[d] = from_f32<T>(to_f32(out[d]) + nonfinite_sum<T>(p, b, kh, d, bad));
    }
  } else if (warp == kScoreWarp) {
    // ---- S = Q K^T ------------------------------------------------------------------
    // The whole warp walks the blocks, so that addresses stay in uniform registers;
    // one lane issues.
    const uint32_t idesc = instruction<T>(kKeys, false);
    const uint32_t q = descriptor(smem_addr(smem)), k0 = descriptor(smem_addr(k_ring));
    int slot = 0, turn = 0;
    bool ready = true;
    for (int k = 0; k < blocks; ++k) {
      const int buffer = k & 1;
      // the products that read this buffer's P, then the keys
      ready = k < 2 || wait_phase(&sh.pv_done[buffer], (k - 2) >> 1 & 1, p.status);
      ready = ready && wait_phase(&sh.k_full[slot], turn, p.status);
      if (!__all_sync(kFullMask, ready)) break;
      fence_after();
      fence_async_proxy();  // the copies are visible to this thread; now to its products
      const uint32_t kd = k0 + slot * (Shape::plane_bytes >> 4);
      const uint32_t d = tmem + Shape::column_s + buffer * kKeys;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kDim / 16; ++kk)
          mma_shared<kDim>(d, q + ((kk / 4 * kPanel + kk % 4 * 32) >> 4),
                           kd + ((kk / 4 * kPanel + kk % 4 * 32) >> 4), idesc, kk > 0);
        commit(&sh.s_full[buffer]);
        mbar_arrive(&sh.s_full[buffer]);
        if (k + Shape::k_stages < blocks) commit(&sh.k_free[slot]);  // else nobody waits for it
      }
      __syncwarp();
      if (++slot == Shape::k_stages) {
        slot = 0;
        turn ^= 1;
      }
    }
    // The softmax warps see the last block's products done; with the one before it, too, no
    // arrival of a product is left that could come after the block has ended.
    if (blocks > 1 && __all_sync(kFullMask, ready))
      wait_phase(&sh.pv_done[blocks & 1], (blocks - 2) >> 1 & 1, p.status);
  } else {
    // ---- O += P V -------------------------------------------------------------------
    const uint32_t idesc = instruction<T>(kDim, true), v0 = descriptor(smem_addr(v_ring));
    int slot = 0, turn = 0;
    for (int k = 0; k < blocks; ++k) {
      const int buffer = k & 1;
      bool ready = wait_phase(&sh.v_full[slot], turn, p.status);
      ready = ready && wait_phase(&sh.p_full[buffer], k >> 1 & 1, p.status);
      if (!__all_sync(kFullMask, ready)) break;
      fence_after();
      fence_async_proxy();
      const uint32_t vd = v0 + slot * (Shape::plane_bytes >> 4);
      const uint32_t weights = tmem + Shape::column_s + buffer * kKeys + kKeys / 2;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          mma_tmem<kDim>(tmem, weights + kk * 8, vd + (kk * 2 * Shape::atom >> 4), idesc,
                         k > 0 || kk > 0);
        commit(&sh.pv_done[buffer]);
        mbar_arrive(&sh.pv_done[buffer]);  // sh.bad reaches the softmax warps by this one
        if (k + Shape::v_stages < blocks) commit(&sh.v_free[slot]);
      }
      __syncwarp();
      if (++slot == Shape::v_stages) {
        slot = 0;
        turn ^= 1;
      }
    }
  }
  __syncwarp();
  fence_before();
  asm volatile("bar.sync 2, %0;\n" ::"n"(32 * (kSoftmaxWarps + 2)) : "memory");
  if (warp == kOutputWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem),
                 "r"(Shape::columns));
  }
}

// The pool as 8-row groups of 64-element panels: (element, row of the group, panel,
// group). Groups are whole where page_size is a multiple of 8. False when the driver
// has no encoder or refuses the sizes: then all rows go through cp.async.
bool encode_pool(CUtensorMap *map, const TreeParams &p, int dtype) {
  using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                              const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<void *> found{nullptr};
  void *fn = found.load(std::memory_order_relaxed);
  if (fn == nullptr) {
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &result) !=
            cudaSuccess ||
        result != cudaDriverEntryPointSuccess || fn == nullptr) {
      cudaGetLastError();
      return false;
    }
    found.store(fn, std::memory_order_relaxed);
  }
  const cuuint64_t row_bytes = (cuuint64_t)p.kv_heads * p.head_dim * 2;
  const cuuint64_t groups = (cuuint64_t)p.pool_blocks * 2 * p.page_size / 8;
  if (groups < 2 || groups > 0x7fffffff) return false;
  const cuuint64_t dims[4] = {64, 8, (cuuint64_t)p.kv_heads * p.head_dim / 64, groups};
  const cuuint64_t strides[3] = {row_bytes, 128, 8 * row_bytes};
  const cuuint32_t box[4] = {64, 8, (cuuint32_t)p.head_dim / 64, kRun / 8}, ones[4] = {1, 1, 1, 1};
  return reinterpret_cast<Encode>(fn)(
             map, dtype == HS_FLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
             4, const_cast<void *>(p.pool), dims, strides, box, ones,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int kDim> int launch(const TreeParams &p, int dtype, cudaStream_t s) {
  auto kernel = tree_tensor_kernel<T, kDim>;
  const size_t bytes = TensorShape<kDim>::dynamic;
  if (int e = reserve_smem(reinterpret_cast<const void *>(kernel), bytes, "attend_tree")) return e;
  const int64_t tiles = ceil_div((int64_t)p.nodes * p.groups, kTile);
  // heads side by side: their slices of a cache row are neighbours in memory
  const dim3 grid((unsigned)(p.kv_heads * tiles), (unsigned)p.splits, (unsigned)p.batch);
  CUtensorMap map{};
  const bool tiled = p.head_dim == kDim && p.count >= kRun && p.page_size % kRun == 0 &&
                     p.page_shift >= 0 && encode_pool(&map, p, dtype);
  kernel<<<grid, kTensorThreads, bytes, s>>>(p, map, tiled);
  return check_launch("tree_tensor_kernel");
}

template <typename T> int launch(const TreeParams &p, int dtype, cudaStream_t s) {
  if (p.head_dim <= 64) return launch<T, 64>(p, dtype, s);
  return p.head_dim <= 128 ? launch<T, 128>(p, dtype, s) : launch<T, 256>(p, dtype, s);
}

}  // namespace

int launch_tree_tensor(const TreeParams &p, int dtype, cudaStream_t s) {
  return dtype == HS_FLOAT16 ? launch<__half>(p, dtype, s) : launch<__nv_bfloat16>(p, dtype, s);
}

}  // namespace hs
