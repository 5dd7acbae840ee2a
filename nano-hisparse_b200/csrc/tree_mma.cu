#include "tree.cuh"

namespace hs {
namespace {

// ---- 16-bit types on the tensor cores ----------------------------------------------------
// 8 warps as kWarpsM x kWarpsN: a warp owns 16 query rows (their fragments of Q
// stay in registers) and 1 / kWarpsN of each stage's keys; warps of the same rows
// join their (O, m, l) at the end. Keys arrive through a ring of kMmaStages
// cp.async stages, 16 bytes a thread, in 16-byte chunks XOR-swizzled by row so
// that ldmatrix meets no bank conflict; the row numbers of a stage are read one
// stage ahead of its copies.
//   S = Q K^T   m16n8k16, K fragments by ldmatrix
//   softmax     fp32 in powers of two; the running maximum is raised only when a
//               score passes it by more than 8 (a factor of 256, far inside
//               fp32 and within fp16's range for P), so O is rescaled rarely
//   O += P V    P rounded to the 16-bit type (a relative error of half a step of
//               each weight, as large as the rounding of the result), V fragments
//               by ldmatrix.trans
// A node's V is copied through registers and its non-finite elements become 0 in
// shared memory: nodes that do not see it would meet 0 * NaN in the product. The
// nodes that do see it get the element added at the end.
constexpr int kMmaThreads = 256;
constexpr int kMmaWarps = kMmaThreads / 32;
constexpr int kMmaStages = 3;
constexpr unsigned char kPlain = 64, kNothing = 65;  // a key's kind: node 0..63, or these

__device__ __forceinline__ void tree_ldmatrix(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tree_ldmatrix_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void tree_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void tree_mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void tree_mma<__half>(float (&c)[4], const uint32_t (&a)[4],
                                                 uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// kDim: head_dim rounded up to the tile (the rest is zero); kWarpsM: 2, 4, 8
template <int kDim, int kWarpsM> struct MmaTile {
  static constexpr int warps_n = kMmaWarps / kWarpsM;
  static constexpr int rows = 16 * kWarpsM;
  static constexpr int stage_keys = 64;
  static constexpr int warp_keys = stage_keys / warps_n;    // 16, 32, 64
  static constexpr int sub_keys = warp_keys < 32 ? warp_keys : 32;
  static constexpr int pitch = kDim * 2;                    // bytes
  static constexpr int stage_bytes = 2 * stage_keys * pitch;
  static constexpr int q_bytes = rows * pitch;
  static constexpr int ring_bytes = kMmaStages * stage_bytes;
  static constexpr int join_pitch = kDim + 4;               // floats
  static constexpr int join_bytes = kMmaWarps * 16 * join_pitch * 4;
  static constexpr size_t bytes =
      q_bytes + (ring_bytes > join_bytes ? ring_bytes : join_bytes) + kMmaStages * stage_keys;
  // blocks on an SM (228 KB, of which every block costs 1 KB besides its own)
  static constexpr int resident = 2 * (bytes + 1280) <= 228 * 1024 ? 2 : 1;
};

template <typename T, int kDim, int kWarpsM>
__global__ void __launch_bounds__(kMmaThreads, (MmaTile<kDim, kWarpsM>::resident))
    tree_mma_kernel(TreeParams p) {
  using Tile = MmaTile<kDim, kWarpsM>;
  constexpr int pitch = Tile::pitch, keys = Tile::stage_keys, chunks = kDim / 8;
  constexpr int row_step = kMmaThreads / chunks, row_loads = keys / row_step;
  constexpr int sub = Tile::sub_keys, nt = sub / 8;  // n-tiles of a sub-tile of scores
  extern __shared__ __align__(128) unsigned char tree_smem[];
  unsigned char *sq = tree_smem, *ring = sq + Tile::q_bytes;
  unsigned char *kinds = tree_smem + Tile::bytes - kMmaStages * keys;
  __shared__ unsigned long long s_bad;  // nodes whose V held a non-finite element
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp % kWarpsM, wn = warp / kWarpsM, split = blockIdx.x;
  const int tiles = (int)ceil_div(p.nodes * p.groups, Tile::rows);
  const int kh = blockIdx.y / tiles, r0 = blockIdx.y % tiles * Tile::rows, b = blockIdx.z;
  const int D = p.head_dim, G = p.groups;
  const int n_nodes = nodes_of(p, b), live = n_nodes * G;
  const int64_t valid = rows_of(p, b);
  const int64_t total = r0 < live ? valid + n_nodes : 0;
  const int64_t chunk = ceil_div(ceil_div(total, p.splits), keys) * keys;
  const int64_t begin = min(total, split * chunk), end = min(total, begin + chunk);
  const int steps = (int)ceil_div(end - begin, keys);
  if (tid == 0) s_bad = 0;

  const int64_t row_elems = (int64_t)p.kv_heads * D;
  const int64_t plane = p.page_size * row_elems;
  const int c = tid % chunks, k_first = tid / chunks;
  const bool in_dim = c * 8 < D;
  const T *pool = static_cast<const T *>(p.pool) + (int64_t)kh * D + c * 8;
  const int64_t node_base = (int64_t)b * p.kv_batch_stride + (int64_t)kh * D + c * 8;
  const T *key = static_cast<const T *>(p.key) + node_base;
  const T *value = static_cast<const T *>(p.value) + node_base;
  const int64_t *rows = p.rows + b * p.rows_batch_stride;

  // the row numbers of a stage's keys that this thread copies a chunk of
  int64_t ahead[row_loads];
  auto look = [&](int step) {
#pragma unroll
    for (int i = 0; i < row_loads; ++i) {
      const int64_t at = begin + (int64_t)step * keys + k_first + i * row_step;
      ahead[i] = at < end && at < valid ? __ldg(rows + at) : -1;
    }
  };
  auto issue = [&](int step) {
    const int slot = step % kMmaStages;
    unsigned char *stage = ring + slot * Tile::stage_bytes;
#pragma unroll
    for (int i = 0; i < row_loads; ++i) {
      const int k = k_first + i * row_step;
      const int64_t at = begin + (int64_t)step * keys + k;
      const uint32_t place = k * pitch + ((c ^ (k & 7)) << 4);
      if (at >= valid && at < end) {  // a node
        const int j = (int)(at - valid);
        uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
        if (in_dim) {
          kx = *reinterpret_cast<const uint4 *>(key + j * p.kv_node_stride);
          vx = *reinterpret_cast<const uint4 *>(value + j * p.kv_node_stride);
        }
        if (clear_nonfinite<T>(vx)) atomicOr(&s_bad, 1ull << j);
        *reinterpret_cast<uint4 *>(stage + place) = kx;
        *reinterpret_cast<uint4 *>(stage + keys * pitch + place) = vx;
        if (c == 0) kinds[slot * keys + k] = (unsigned char)j;
      } else {
        const int64_t off = row_offset(p, ahead[i], row_elems);
        const bool ok = off >= 0;
        const T *src = ok ? pool + off : pool;
        tree_cp_async16(smem_addr(stage + place), src, ok && in_dim);
        tree_cp_async16(smem_addr(stage + keys * pitch + place), ok ? src + plane : src,
                        ok && in_dim);
        if (c == 0) kinds[slot * keys + k] = ok ? kPlain : kNothing;
      }
    }
  };
  if (steps > 0) look(0);
  __syncthreads();  // s_bad
#pragma unroll
  for (int s = 0; s < kMmaStages - 1; ++s) {
    if (s < steps) {
      issue(s);
      look(s + 1);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  }

  // Q: rows r0 .., zero beyond the last
  const T *query = static_cast<const T *>(p.query) + b * p.q_batch_stride;
  for (int i = tid; i < Tile::rows * chunks; i += kMmaThreads) {
    const int r = i / chunks, qc = i % chunks, row = r0 + r;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (row < live && qc * 8 < D)
      x = *reinterpret_cast<const uint4 *>(query + row / G * p.q_node_stride +
                                           (int64_t)(kh * G + row % G) * D + qc * 8);
    *reinterpret_cast<uint4 *>(sq + r * pitch + ((qc ^ (r & 7)) << 4)) = x;
  }
  __syncthreads();
  // lane's two rows, and what their nodes see
  const int row_lo = r0 + wm * 16 + lane / 4, row_hi = row_lo + 8;
  uint64_t see_lo = 0, see_hi = 0;
  if (row_lo < live) see_lo = (uint64_t)p.mask[(int64_t)b * p.nodes + row_lo / G];
  if (row_hi < live) see_hi = (uint64_t)p.mask[(int64_t)b * p.nodes + row_hi / G];

  constexpr bool q_in_registers = kDim <= 128;
  uint32_t qf[q_in_registers ? kDim / 16 : 1][4];
  const int q_row = wm * 16 + (lane & 15);
  auto load_q = [&](int kk, uint32_t (&f)[4]) {
    tree_ldmatrix(smem_addr(sq + q_row * pitch + (((2 * kk + (lane >> 4)) ^ (q_row & 7)) << 4)),
                  f);
  };
  if constexpr (q_in_registers)
#pragma unroll
    for (int kk = 0; kk < kDim / 16; ++kk) load_q(kk, qf[kk]);

  float o[kDim / 8][4];
#pragma unroll
  for (int j = 0; j < kDim / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
  float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;

  for (int step = 0; step < steps; ++step) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kMmaStages - 2) : "memory");
    __syncthreads();
    if (step + kMmaStages - 1 < steps) {
      issue(step + kMmaStages - 1);
      look(step + kMmaStages);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    const int slot = step % kMmaStages;
    const unsigned char *sk = ring + slot * Tile::stage_bytes, *sv = sk + keys * pitch;
#pragma unroll
    for (int part = 0; part < Tile::warp_keys / sub; ++part) {
      const int k0 = wn * Tile::warp_keys + part * sub;
      float s[nt][4];
#pragma unroll
      for (int j = 0; j < nt; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < kDim / 16; ++kk) {
        uint32_t af[4];
        if constexpr (q_in_registers) {
#pragma unroll
          for (int e = 0; e < 4; ++e) af[e] = qf[kk][e];
        } else {
          load_q(kk, af);
        }
#pragma unroll
        for (int j = 0; j < nt; j += 2) {
          // keys 8 j .. 8 j + 15: lanes 0-7 rows 0-7 low half, 8-15 its high half, then rows 8-15
          const int kr = k0 + j * 8 + (lane & 7) + ((lane >> 4) << 3);
          const int kc = 2 * kk + ((lane >> 3) & 1);
          uint32_t kf[4];
          tree_ldmatrix(smem_addr(sk + kr * pitch + ((kc ^ (kr & 7)) << 4)), kf);
          tree_mma<T>(s[j], af, kf[0], kf[1]);
          tree_mma<T>(s[j + 1], af, kf[2], kf[3]);
        }
      }
      // what each score's key is: two keys a 16-bit word
      bool plain = true;
      unsigned kind[nt];
#pragma unroll
      for (int j = 0; j < nt; ++j) {
        kind[j] = *reinterpret_cast<const unsigned short *>(
            kinds + slot * keys + k0 + j * 8 + (lane & 3) * 2);
        plain = plain && kind[j] == (kPlain | kPlain << 8);
      }
      float top_lo = -INFINITY, top_hi = -INFINITY;
#pragma unroll
      for (int j = 0; j < nt; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] *= p.scale_log2;
        if (!plain) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const unsigned kd = kind[j] >> (8 * e) & 0xff;
            if (kd == kNothing || (kd < kPlain && !(see_lo >> kd & 1))) s[j][e] = -INFINITY;
            if (kd == kNothing || (kd < kPlain && !(see_hi >> kd & 1))) s[j][2 + e] = -INFINITY;
          }
        }
        top_lo = fmaxf(top_lo, fmaxf(s[j][0], s[j][1]));
        top_hi = fmaxf(top_hi, fmaxf(s[j][2], s[j][3]));
      }
      const bool raise = top_lo > m_lo + kLazy || top_hi > m_hi + kLazy;
      if (__any_sync(kFullMask, raise)) {
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {
          top_lo = fmaxf(top_lo, __shfl_xor_sync(kFullMask, top_lo, d));
          top_hi = fmaxf(top_hi, __shfl_xor_sync(kFullMask, top_hi, d));
        }
        const float new_lo = fmaxf(m_lo, top_lo), new_hi = fmaxf(m_hi, top_hi);
        const float f_lo = m_lo == -INFINITY ? 0.f : tree_exp2(m_lo - new_lo);
        const float f_hi = m_hi == -INFINITY ? 0.f : tree_exp2(m_hi - new_hi);
        m_lo = new_lo;
        m_hi = new_hi;
        l_lo *= f_lo;
        l_hi *= f_hi;
#pragma unroll
        for (int j = 0; j < kDim / 8; ++j) {
          o[j][0] *= f_lo;
          o[j][1] *= f_lo;
          o[j][2] *= f_hi;
          o[j][3] *= f_hi;
        }
      }
      // a row that has seen nothing keeps m = -inf: its weights are exp2(-inf) = 0
      const float b_lo = m_lo == -INFINITY ? 0.f : m_lo - kLift<T>;
      const float b_hi = m_hi == -INFINITY ? 0.f : m_hi - kLift<T>;
#pragma unroll
      for (int j = 0; j < nt; ++j) {
        s[j][0] = tree_exp2(s[j][0] - b_lo);
        s[j][1] = tree_exp2(s[j][1] - b_lo);
        s[j][2] = tree_exp2(s[j][2] - b_hi);
        s[j][3] = tree_exp2(s[j][3] - b_hi);
        l_lo += s[j][0] + s[j][1];
        l_hi += s[j][2] + s[j][3];
      }
#pragma unroll
      for (int kk = 0; kk < sub / 16; ++kk) {
        const uint32_t pf[4] = {pack2<T>(s[2 * kk][0], s[2 * kk][1]),
                                pack2<T>(s[2 * kk][2], s[2 * kk][3]),
                                pack2<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                                pack2<T>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
        const int vr = k0 + kk * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < kDim / 8; j += 2) {
          uint32_t vf[4];
          tree_ldmatrix_trans(
              smem_addr(sv + vr * pitch + (((j + (lane >> 4)) ^ (vr & 7)) << 4)), vf);
          tree_mma<T>(o[j], pf, vf[0], vf[1]);
          tree_mma<T>(o[j + 1], pf, vf[2], vf[3]);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
  for (int d = 1; d <= 2; d <<= 1) {
    l_lo += __shfl_xor_sync(kFullMask, l_lo, d);
    l_hi += __shfl_xor_sync(kFullMask, l_hi, d);
  }
  // join the warps of the same rows through the ring's memory
  __syncthreads();
  float *join = reinterpret_cast<float *>(ring);
  constexpr int jp = Tile::join_pitch;
  {
    float *lo = join + (warp * 16 + lane / 4) * jp, *hi = lo + 8 * jp;
#pragma unroll
    for (int j = 0; j < kDim / 8; ++j) {
      const int d = j * 8 + (lane & 3) * 2;
      *reinterpret_cast<float2 *>(lo + d) = make_float2(o[j][0], o[j][1]);
      *reinterpret_cast<float2 *>(hi + d) = make_float2(o[j][2], o[j][3]);
    }
    if ((lane & 3) == 0) {
      lo[kDim] = m_lo;
      lo[kDim + 1] = l_lo;
      hi[kDim] = m_hi;
      hi[kDim + 1] = l_hi;
    }
  }
  __syncthreads();
  const unsigned long long bad = s_bad;
  T *out = static_cast<T *>(p.out) + (int64_t)b * p.nodes * p.q_heads * D;
  const int rows_here = min(Tile::rows, p.nodes * G - r0);
  for (int r = warp; r < rows_here; r += kMmaWarps) {
    const int row = r0 + r;
    const float *first = join + (r / 16 * 16 + r % 16) * jp;  // warp r / 16 of column wn = 0
    float m = -INFINITY, l = 0.f, w[Tile::warps_n];
#pragma unroll
    for (int k = 0; k < Tile::warps_n; ++k) m = fmaxf(m, first[k * kWarpsM * 16 * jp + kDim]);
#pragma unroll
    for (int k = 0; k < Tile::warps_n; ++k) {
      const float mk = first[k * kWarpsM * 16 * jp + kDim];
      w[k] = mk == -INFINITY ? 0.f : tree_exp2(mk - m);
      l += first[k * kWarpsM * 16 * jp + kDim + 1] * (mk == -INFINITY ? 1.f : w[k]);
    }
    const uint64_t see = bad != 0 && row < live ? (uint64_t)p.mask[(int64_t)b * p.nodes + row / G] : 0;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    for (int d = lane; d < D; d += 32) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < Tile::warps_n; ++k) x = fmaf(first[k * kWarpsM * 16 * jp + d], w[k], x);
      if ((bad & see) != 0) x += nonfinite_sum<T>(p, b, kh, d, bad & see);
      if (p.splits == 1)
        out[(int64_t)(row / G) * p.q_heads * D + (int64_t)(kh * G + row % G) * D + d] =
            from_f32<T>(row < live ? x * inv : 0.f);
      else
        reinterpret_cast<float *>(quad_of(p, part_of(p, b, kh, split), row, d / 4))[d % 4] = x;
    }
    if (p.splits > 1 && lane == 0)
      *stat_of(p, part_of(p, b, kh, split), row) = make_float2(m, l);
  }
}

template <typename T, int kWarpsM> int launch(const TreeParams &p, cudaStream_t s) {
  using Tile = MmaTile<256, kWarpsM>;
  auto kernel = tree_mma_kernel<T, 256, kWarpsM>;
  if (int e = reserve_smem(reinterpret_cast<const void *>(kernel), Tile::bytes, "attend_tree"))
    return e;
  const int64_t tiles = ceil_div((int64_t)p.nodes * p.groups, Tile::rows);
  const dim3 grid((unsigned)p.splits, (unsigned)(p.kv_heads * tiles), (unsigned)p.batch);
  kernel<<<grid, kMmaThreads, Tile::bytes, s>>>(p);
  return check_launch("tree_mma_kernel");
}

}  // namespace

int launch_tree_mma(const TreeParams &p, int dtype, cudaStream_t s) {
  if (dtype == HS_FLOAT16) return p.tile_rows == 32 ? launch<__half, 2>(p, s) : launch<__half, 4>(p, s);
  return p.tile_rows == 32 ? launch<__nv_bfloat16, 2>(p, s) : launch<__nv_bfloat16, 4>(p, s);
}

}  // namespace hs
