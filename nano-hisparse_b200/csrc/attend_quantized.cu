// (11) Decode attention over the rows of an 8-bit cache.
//
// s_i = (q . k_i) 2^ek_i / sqrt(head_dim) with k_i the codes, in powers of two. A row's V
// scale goes into its weight, so that the codes are multiplied as they are: with m the
// running maximum of s_i + ev_i,
//   o += 2^(s_i + ev_i - m) v_i     l += 2^(s_i - m + kSumLift)     out = o / l 2^kSumLift
// The two powers are taken apart: a row with a small scale may weigh nothing in o and
// most in l. As scales are 2^-100 to 2^120, the largest term of l lies between 2^-110 and
// 2^110, and l stays inside fp32: on CUDA cores a block has at most 2^17 rows (of requests of up
// to 2^24; it takes that many of zeros to make the sum too large), on tensor cores a large
// sum is lowered. The maximum is kept as its row's score and exponent, whose
// rounded sum would cost digits of the weights.
#include "attend_quantized.cuh"

namespace hs {
namespace {

constexpr int kSimtThreads = 128;
constexpr int kSimtWarps = kSimtThreads / 32;
constexpr int kSimtHeads = 8;    // query heads of a block
constexpr int kSimtAhead = 4;    // rows of a warp in flight

// CUDA cores, every type and shape: rows of their own for each query head, head_dims that
// are no multiple of 16. A warp takes four rows at a time, a lane C neighbouring elements of
// each. Its reads by the byte and a shuffle tree for each score bound it: 16 requests of
// 2,048 rows, 32/8 heads of 128, take 213 us, 18 on tensor cores. kCluster: a request's splits
// are a cluster that joins them, without a workspace (simt_splits).
template <typename T, int C, bool kCluster>
__global__ void __launch_bounds__(kSimtThreads) quant_simt_kernel(QuantAttendParams p) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  __shared__ float4 red[kSimtWarps][kSimtHeads];  // a maximum's score, exponent; the sum
  __shared__ float red_o[kSimtWarps][kSimtHeads][32 * C];
  __shared__ float4 block_stats[kSimtHeads];  // of all warps
  const int split = blockIdx.x, b = blockIdx.z, D = p.head_dim;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d0 = lane * C;
  int kh, h0, hn;
  if (p.rows_head_stride == 0) {
    const int chunks = (p.groups + kSimtHeads - 1) / kSimtHeads;
    kh = blockIdx.y / chunks;
    h0 = kh * p.groups + blockIdx.y % chunks * kSimtHeads;
    hn = min(kSimtHeads, (kh + 1) * p.groups - h0);
  } else {
    h0 = blockIdx.y;
    kh = h0 / p.groups;
    hn = 1;
  }
  float q[kSimtHeads][C], ms[kSimtHeads], me[kSimtHeads], l[kSimtHeads], o[kSimtHeads][C];
  const T *query = static_cast<const T *>(p.query) + (int64_t)b * p.q_batch_stride;
#pragma unroll
  for (int g = 0; g < kSimtHeads; ++g) {
    ms[g] = -INFINITY;
    me[g] = l[g] = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      q[g][c] = g < hn && d0 + c < D ? to_f32(query[(int64_t)(h0 + g) * D + d0 + c]) : 0.f;
      o[g][c] = 0.f;
    }
  }
  const int64_t valid = quant_rows(p, b), share = ceil_div(valid, p.splits);
  const int64_t begin = min(valid, split * share), end = min(valid, begin + share);
  const int64_t *rows = p.rows + b * p.rows_batch_stride + h0 * p.rows_head_stride;
  const int64_t E = (int64_t)p.kv_heads * D, plane = (int64_t)p.page_size * p.record;
  for (int64_t i0 = begin + warp * kSimtAhead; i0 < end; i0 += kSimtWarps * kSimtAhead) {
    float k[kSimtAhead][C], v[kSimtAhead][C], k_scale[kSimtAhead];
    int v_exponent[kSimtAhead];
    bool seen[kSimtAhead];
#pragma unroll
    for (int r = 0; r < kSimtAhead; ++r) {
      const int64_t index = i0 + r < end ? record_index(rows[i0 + r], p.page_size, p.page_shift,
                                                        p.pool_blocks, p.status) : -1;
      seen[r] = index >= 0 && p.pool[index * p.record + E + kh] != 0;
      k_scale[r] = 0.f;
      v_exponent[r] = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) k[r][c] = v[r][c] = 0.f;
      if (!seen[r]) continue;
      const unsigned char *record = p.pool + index * p.record;
      k_scale[r] = scale_of(record[E + kh]) * p.scale_log2;
      v_exponent[r] = (int)record[plane + E + kh] - 127;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (d0 + c < D) {
          k[r][c] = decode1(record[(int64_t)kh * D + d0 + c]);
          v[r][c] = decode1(record[plane + (int64_t)kh * D + d0 + c]);
        }
    }
#pragma unroll
    for (int r = 0; r < kSimtAhead; ++r) {
      if (!seen[r]) continue;  // the same for the whole warp
#pragma unroll
      for (int g = 0; g < kSimtHeads; ++g) {
        if (g >= hn) break;
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) dot = fmaf(q[g][c], k[r][c], dot);
        const float s = warp_xor_tree_sum(dot) * k_scale[r], e = (float)v_exponent[r];
        if (ms[g] == -INFINITY || s + e > ms[g] + me[g]) {  // the new maximum (or NaN, kept)
          const float f = ms[g] == -INFINITY ? 0.f : quant_share(ms[g], me[g], s, e);
          l[g] *= f;
#pragma unroll
          for (int c = 0; c < C; ++c) o[g][c] *= f;
          ms[g] = s;
          me[g] = e;
        }
        const float w = quant_share(s, e, ms[g], me[g]);
        l[g] += quant_share(s, kSumLift, ms[g], me[g]);
#pragma unroll
        for (int c = 0; c < C; ++c) o[g][c] = fmaf(w, v[r][c], o[g][c]);
      }
    }
  }
  const auto write = [&](int g, int d, float x, float sum) {
    const float y = sum > 0.f || sum != sum ? x / sum * kSumScale : 0.f;
    static_cast<T *>(p.out)[((int64_t)b * p.q_heads + h0 + g) * D + d] = from_f32<T>(y);
  };
  // the warps' results
#pragma unroll
  for (int g = 0; g < kSimtHeads; ++g) {
    if (g >= hn) break;
    if (lane == 0) red[warp][g] = make_float4(ms[g], me[g], l[g], 0.f);
#pragma unroll
    for (int c = 0; c < C; ++c) red_o[warp][g][d0 + c] = o[g][c];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < hn * 32 * C; i += kSimtThreads) {
    const int g = i / (32 * C), d = i % (32 * C);
    if (d >= D) continue;
    float4 top = red[0][g];
    float sum = 0.f, x = 0.f;
    for (int w = 1; w < kSimtWarps; ++w) top = quant_larger(top, red[w][g]);
    for (int w = 0; w < kSimtWarps; ++w) {
      const float4 part = red[w][g];
      if (part.z == 0.f) continue;  // saw nothing
      const float f = quant_share(part.x, part.y, top.x, top.y);
      sum = fmaf(part.z, f, sum);
      x = fmaf(red_o[w][g][d], f, x);
    }
    if constexpr (kCluster) {
      if (d == 0) block_stats[g] = make_float4(top.x, top.y, sum, 0.f);
      red_o[0][g][d] = x;  // read by this thread alone so far
    } else if (p.out != nullptr) {
      write(g, d, x, sum);
    } else {
      const int64_t part = quant_part(p, p.phase, b, h0 + g, split);
      if (d == 0) p.stats[part] = make_float4(top.x, top.y, sum, 0.f);
      p.partials[part * quant_pad(D) + d] = x;
    }
  }
  if constexpr (!kCluster) return;
  // the splits' results; every thread of the cluster comes to both barriers
  cluster_barrier();
  for (int i = split * kSimtThreads + threadIdx.x; i < hn * 32 * C;
       i += p.splits * kSimtThreads) {
    const int g = i / (32 * C), d = i % (32 * C);
    if (d >= D) continue;
    float4 top = *map_rank(&block_stats[g], 0);
    float sum = 0.f, x = 0.f;
    for (int k = 1; k < p.splits; ++k) top = quant_larger(top, *map_rank(&block_stats[g], k));
    for (int k = 0; k < p.splits; ++k) {
      const float4 part = *map_rank(&block_stats[g], k);
      if (part.z == 0.f) continue;  // saw nothing
      const float f = quant_share(part.x, part.y, top.x, top.y);
      sum = fmaf(part.z, f, sum);
      x = fmaf(*map_rank(&red_o[0][g][d], k), f, x);
    }
    write(g, d, x, sum);
  }
  cluster_barrier();  // the others may still read this block's results
}

// ---- the join of splits and phases ----------------------------------------------------------
constexpr int kJoinThreads = 256, kJoinAhead = 4;

// One block a query head. A thread reads the statistics of one partial result (at most two
// phases of kQuantMaxSplits), whose weights meet in shared memory; then kLanes threads
// have four elements each, and kJoinThreads / kLanes groups of them a share of the
// results, kJoinAhead loads in flight. Its launch overlaps the end of the kernel before it;
// latencies bound what is left, 2.5 to 5 us for 9 to 128 splits.
template <typename T, int kLanes>
__global__ void __launch_bounds__(kJoinThreads) quant_merge_kernel(QuantAttendParams p, int phases,
                                                                   T *out) {
  constexpr int kGroups = kJoinThreads / kLanes, kWarps = kJoinThreads / 32;
  static_assert(2 * kQuantMaxSplits <= kJoinThreads, "a thread for each partial result");
  __shared__ float weights[kJoinThreads];
  __shared__ float4 tops[kWarps];
  __shared__ float totals[kWarps];
  __shared__ float4 sums[kGroups][kLanes];
  const int h = blockIdx.x, b = blockIdx.y, D = p.head_dim, quads = quant_pad(D) / 4;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, all = phases * p.splits;
  const int quad = tid % kLanes, group = tid / kLanes;
  const auto part = [&](int i) {
    const int phase = i >= p.splits;
    return quant_part(p, phase, b, h, i - phase * p.splits);
  };
  const auto load = [&](int i, float4(&x)[kJoinAhead]) {
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u)
      if (i + u * kGroups < all && quad < quads)
        x[u] = reinterpret_cast<const float4 *>(p.partials)[part(i + u * kGroups) * quads + quad];
  };
  // Every thread waits: this kernel must not end before the one that writes the workspace.
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  float4 x[kJoinAhead];
  const float4 mine = tid < all ? p.stats[part(tid)] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
  load(group, x);
  float4 top = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    top = quant_larger(top, make_float4(__shfl_xor_sync(kFullMask, top.x, o),
                                        __shfl_xor_sync(kFullMask, top.y, o),
                                        __shfl_xor_sync(kFullMask, top.z, o), 0.f));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = quant_larger(top, tops[w]);
  // one that saw nothing left no output: below 0
  const float f = mine.z == 0.f ? -1.f : quant_share(mine.x, mine.y, top.x, top.y);
  weights[tid] = f;
  const float share = warp_xor_tree_sum(mine.z == 0.f ? 0.f : mine.z * f);
  if (lane == 0) totals[warp] = share;
  __syncthreads();
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = group; i < all; i += kJoinAhead * kGroups) {
    if (i != group) load(i, x);
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      if (i + u * kGroups >= all) break;
      const float w = weights[i + u * kGroups];
      if (w < 0.f || quad >= quads) continue;
      sum.x = fmaf(w, x[u].x, sum.x);
      sum.y = fmaf(w, x[u].y, sum.y);
      sum.z = fmaf(w, x[u].z, sum.z);
      sum.w = fmaf(w, x[u].w, sum.w);
    }
  }
  sums[group][quad] = sum;
  __syncthreads();
  float l = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) l += totals[w];
  const float inv = l > 0.f || l != l ? kSumScale / l : 0.f;
  if (tid >= D) return;
  float y = 0.f;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) y += reinterpret_cast<const float *>(sums[g])[tid];
  out[((int64_t)b * p.q_heads + h) * D + tid] = from_f32<T>(y * inv);
}

// Splits that leave a block of the CUDA-core kernel at most 2^17 rows: the sum of their weights
// stays inside fp32 whatever the rows hold.
int64_t fewest_splits(int64_t count) {
  const int64_t n = ceil_div(count, (int64_t)1 << 17);
  return n < kQuantMaxSplits ? n : kQuantMaxSplits;
}
// Splits that a call in one phase may have without a join and without a workspace: those of
// a cluster, for the tensor-core kernel's head_dims and two blocks an SM (with one, clusters
// leave SMs idle: 4 requests of 4,096 rows, one head of 256: 22.7 us as a cluster of 8, 17.1
// with a join). A call without a join that cannot take that kernel has simt_splits.
int splits_without_join(const QuantMmaGrid &g, int head_dim) {
  return head_dim % 16 == 0 && g.resident == 2 ? kClusterSplits : 1;
}
// Splits of a request's rows, from what was measured of the tensor-core kernel, in ns: a
// warp takes 1,450 for a unit of 32 rows (2,500 above head_dim 128) while memory keeps up,
// the blocks of an SM together 1,730 for 67.6 KB of records. A block takes 3,000 besides
// (half of it beside another block's work), one whose warps share a head's rows 250 more for
// each query to join them, and the second kernel 2,500 and 20 for each split. So more blocks
// than one an SM do not help large calls (16 requests of 2,048 rows, 8 heads of 128: 9 splits
// 18.9 us, 18 splits 18.2, 37 splits 22.5), and small ones want a unit a warp (1 of 8,192:
// 64 splits 12.7, 18 splits 26.2) or less where warps share a head (2 of 2,000, one head of
// 256: 4 splits 20.3, 18 splits 14.2). A cluster saves the second launch and its traffic (4
// requests of 1,000 rows: 8 splits 9.5, 10.6 with 9 splits and a join). But its blocks crowd
// on some SMs while others idle: they count for a third more (16 of 2,048: 8 splits 21.5),
// and with much to do only a grid that fills the SMs once takes one (53 of 3,057, 4 heads of
// 128: 5 splits 39.2, 11 splits with a join 47.6; but 16 of 32,768, 8 heads: 8 splits 288, 18
// with a join 168).
int quant_splits(const QuantMmaGrid &g, int batch, int head_dim, int64_t count) {
  const int64_t blocks = (int64_t)batch * g.groups * g.chunks, sms = sm_count();
  const int64_t units = ceil_div(count, 32);
  const int64_t most = units < kQuantMaxSplits ? units : kQuantMaxSplits;
  const int64_t compute = head_dim > 128 ? 2500 : 1450;
  const int64_t share = (int64_t)64 * g.heads * (head_dim + 1) * 1730 / 67584;
  int64_t best = 1, least = 0;
  const auto consider = [&](int64_t n) {
    if (n > most) n = most;
    if (n < 1) n = 1;
    const int64_t own = ceil_div(units, n);  // units of a split
    if (own > 0) n = ceil_div(units, own);   // the fewest such
    const bool join = n > splits_without_join(g, head_dim), cluster = !join && n > 1;
    const int64_t all = blocks * n, beside = all > sms ? g.resident : 1;
    const int64_t rounds = ceil_div(all, beside * sms);
    const int64_t alone = ceil_div(own, g.slices) * compute, shared = own * beside * share;
    int64_t time = rounds * (alone > shared ? alone : shared);
    if (cluster && all <= sms) time = time * 4 / 3;
    if (cluster && time > 15000 && (all <= sms || rounds > 1)) return;
    time += rounds * (g.slices > 1 ? 3000 + 250 * g.queries : 3000 / beside);
    time += join ? 2500 + 20 * n : cluster ? 1000 : 0;
    if (least == 0 || time < least) {
      least = time;
      best = n;
    }
  };
  consider(1);
  consider(4);
  consider(kClusterSplits);
  for (int i = 1; i <= 4; ++i) consider(sms * i / blocks);
  consider(most);
  return (int)(best > fewest_splits(count) ? best : fewest_splits(count));
}

int check_sizes(int batch, int dtype, int64_t pool_blocks, int64_t count, int q_heads,
                int kv_heads, int head_dim, int page_size) {
  if (batch < 0 || kv_heads < 1 || q_heads < 1 || head_dim < 1 || page_size < 1 ||
      pool_blocks < 0 || count < 0)
    return set_error(HS_ERR_INVALID_ARGUMENT, "attend_quantized: invalid sizes");
  if (q_heads % kv_heads)
    return set_error(HS_ERR_INVALID_ARGUMENT, "query GQA/device mismatch");
  if (head_dim > kQuantMaxDim)
    return set_error(HS_ERR_UNSUPPORTED, "attend_quantized: head_dim %d > %d is not supported",
                     head_dim, kQuantMaxDim);
  if (dtype != HS_FLOAT32 && dtype != HS_FLOAT16 && dtype != HS_BFLOAT16)
    return set_error(HS_ERR_INVALID_ARGUMENT, "attend_quantized: invalid dtype %d", dtype);
  if (batch > 65535 || q_heads > 32767 || count > 0x7fffff00)
    return set_error(HS_ERR_UNSUPPORTED, "attend_quantized: batch, heads or rows too many");
  return HS_OK;
}

size_t workspace_of(const QuantAttendParams &p, int phases) {
  const int64_t parts = p.join ? (int64_t)phases * p.batch * p.q_heads * p.splits : 0;
  return (size_t)parts * (sizeof(float4) + quant_pad(p.head_dim) * sizeof(float));
}
// Whether the workspace holds `phases` phases
int check_workspace(const QuantAttendParams &p, int phases, void *workspace, size_t bytes) {
  const size_t need = workspace_of(p, phases);
  if (need == 0) return HS_OK;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0)
    return set_error(HS_ERR_WORKSPACE, "attend_quantized: the workspace must be 16-byte aligned");
  if (!workspace || bytes < need)
    return set_error(HS_ERR_WORKSPACE, "attend_quantized: workspace of %zu bytes < required %zu",
                     bytes, need);
  return HS_OK;
}

// Splits of a call on CUDA cores without a join, as a cluster: while one round of blocks
// takes them all (registers leave an SM four blocks up to head_dim 64, three up to 128, two
// above) and each has 16 rows. Of 32/8 heads of 128 with rows of their own, 200 rows: 1
// request 8 splits 11 us, 1 split 42; 4 requests 2 splits 25, 1 split 42, 8 splits 32;
// 64 requests 1 split 186, 4 splits 260.
int simt_splits(const QuantAttendParams &p) {
  const int per = (p.groups + kSimtHeads - 1) / kSimtHeads;
  const int64_t blocks = (int64_t)p.batch *
                         (p.rows_head_stride == 0 ? p.kv_heads * per : p.q_heads);
  const int64_t places = (int64_t)sm_count() * (p.head_dim <= 64 ? 4 : p.head_dim <= 128 ? 3 : 2);
  int n = kClusterSplits;
  while (n > 1 && (blocks * n > places || (int64_t)n * 16 > p.count + 15) &&
         n / 2 >= fewest_splits(p.count))
    n >>= 1;
  return n;
}
template <typename T, bool kCluster> int launch_rows(const QuantAttendParams &p, cudaStream_t s) {
  const int per = (p.groups + kSimtHeads - 1) / kSimtHeads;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)p.splits,
                        (unsigned)(p.rows_head_stride == 0 ? p.kv_heads * per : p.q_heads),
                        (unsigned)p.batch);
  config.blockDim = dim3(kSimtThreads);
  config.stream = s;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = (unsigned)p.splits;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = kCluster ? 1 : 0;
  switch (ceil_div(p.head_dim, 32)) {
    case 1: cudaLaunchKernelEx(&config, quant_simt_kernel<T, 1, kCluster>, p); break;
    case 2: cudaLaunchKernelEx(&config, quant_simt_kernel<T, 2, kCluster>, p); break;
    case 3:
    case 4: cudaLaunchKernelEx(&config, quant_simt_kernel<T, 4, kCluster>, p); break;
    default: cudaLaunchKernelEx(&config, quant_simt_kernel<T, 8, kCluster>, p); break;
  }
  return check_launch("quant_simt_kernel");
}
template <typename T> int launch_rows(const QuantAttendParams &p, cudaStream_t s) {
  return p.out != nullptr && p.splits > 1 ? launch_rows<T, true>(p, s)
                                          : launch_rows<T, false>(p, s);
}
// beside: whether its launch may overlap the end of the kernel before it, which it waits
// for itself
template <typename T>
int launch_merge(const QuantAttendParams &p, int phases, void *out, bool beside, cudaStream_t s) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)p.q_heads, (unsigned)p.batch);
  config.blockDim = dim3(kJoinThreads);
  config.stream = s;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = beside ? 1 : 0;
  T *to = static_cast<T *>(out);
  if (p.head_dim <= 64) cudaLaunchKernelEx(&config, quant_merge_kernel<T, 16>, p, phases, to);
  else if (p.head_dim <= 128) cudaLaunchKernelEx(&config, quant_merge_kernel<T, 32>, p, phases, to);
  else cudaLaunchKernelEx(&config, quant_merge_kernel<T, 64>, p, phases, to);
  return check_launch("quant_merge_kernel");
}
// Whether the tensor-core kernel takes a call: it reads four query elements together and
// numbers records in 32 bits.
bool on_tensor_cores(const QuantAttendParams &p, int dtype) {
  const int four = dtype == HS_FLOAT32 ? 16 : 8;
  return p.head_dim % 16 == 0 && p.rows_head_stride == 0 &&
         reinterpret_cast<uintptr_t>(p.query) % four == 0 && p.q_batch_stride % 4 == 0 &&
         p.pool_blocks <= 0xfffffffell / 2 / p.page_size;
}
int launch_rows(const QuantAttendParams &p, int dtype, cudaStream_t s) {
  if (on_tensor_cores(p, dtype)) return launch_quant_mma(p, dtype, s);
  switch (dtype) {
    case HS_FLOAT32: return launch_rows<float>(p, s);
    case HS_FLOAT16: return launch_rows<__half>(p, s);
    default: return launch_rows<__nv_bfloat16>(p, s);
  }
}
int launch_merge(const QuantAttendParams &p, int phases, void *out, int dtype, bool beside,
                 cudaStream_t s) {
  switch (dtype) {
    case HS_FLOAT32: return launch_merge<float>(p, phases, out, beside, s);
    case HS_FLOAT16: return launch_merge<__half>(p, phases, out, beside, s);
    default: return launch_merge<__nv_bfloat16>(p, phases, out, beside, s);
  }
}

// The parameters that every form has; the workspace holds `phases` phases.
QuantAttendParams params_of(int batch, int phases, int dtype, int q_heads, int kv_heads,
                            int head_dim, int64_t count, void *workspace) {
  QuantAttendParams p{};
  p.batch = batch;
  p.count = count;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.head_dim = head_dim;
  p.groups = q_heads / kv_heads;
  const QuantMmaGrid g = quant_mma_grid(dtype, q_heads, kv_heads, head_dim);
  p.splits = quant_splits(g, batch, head_dim, count);
  p.join = phases > 1 || p.splits > splits_without_join(g, head_dim);
  p.record = record_bytes(kv_heads, head_dim);
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
  p.stats = static_cast<float4 *>(workspace);
  p.partials = reinterpret_cast<float *>(p.stats + (int64_t)phases * batch * q_heads * p.splits);
  return p;
}

}  // namespace
}  // namespace hs

extern "C" size_t hs_attend_quantized_workspace_bytes(int batch, int phases, int dtype,
                                                      int q_heads, int kv_heads, int head_dim,
                                                      int64_t count) {
  using namespace hs;
  if (batch < 1 || phases < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || count < 0)
    return 0;
  const QuantAttendParams p =
      params_of(batch, phases, dtype, q_heads, kv_heads, head_dim, count, nullptr);
  return workspace_of(p, phases);
}

extern "C" int hs_attend_quantized(int batch, const void *query, int64_t query_batch_stride,
                                   int dtype, const void *pool, int64_t pool_blocks,
                                   const int64_t *rows, int64_t rows_batch_stride,
                                   int64_t rows_head_stride, int64_t count, const int32_t *counts,
                                   void *out, int q_heads, int kv_heads, int head_dim,
                                   int page_size, void *workspace, size_t workspace_bytes,
                                   int32_t *device_status, hs_stream stream) {
  using namespace hs;
  if (int e = check_sizes(batch, dtype, pool_blocks, count, q_heads, kv_heads, head_dim,
                          page_size))
    return e;
  if (batch == 0) return HS_OK;
  if (!query || !out || (count > 0 && (!rows || !pool)))
    return set_error(HS_ERR_INVALID_ARGUMENT, "attend_quantized: null pointer");
  if ((reinterpret_cast<uintptr_t>(pool) & 15) != 0)
    return set_error(HS_ERR_INVALID_ARGUMENT,
                     "attend_quantized: the pool must be 16-byte aligned");
  QuantAttendParams p = params_of(batch, 1, dtype, q_heads, kv_heads, head_dim, count, workspace);
  if (int e = check_workspace(p, 1, workspace, workspace_bytes)) return e;
  p.query = query;
  p.q_batch_stride = query_batch_stride;
  p.pool = static_cast<const unsigned char *>(pool);
  p.pool_blocks = pool_blocks;
  p.rows = rows;
  p.rows_batch_stride = rows_batch_stride;
  p.rows_head_stride = rows_head_stride;
  p.counts32 = counts;
  p.page_size = page_size;
  p.page_shift = page_shift_of(page_size);
  p.status = device_status;
  if (!p.join) {
    p.out = out;
    if (!on_tensor_cores(p, dtype)) p.splits = simt_splits(p);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int status = launch_rows(p, dtype, s);
  return status != HS_OK || p.out != nullptr ? status : launch_merge(p, 1, out, dtype, true, s);
}

extern "C" int hs_attend_quantized_phase(int batch, const void *query,
                                         int64_t query_batch_stride, int dtype, const void *pool,
                                         int64_t pool_blocks, const int64_t *rows,
                                         int64_t rows_batch_stride, int64_t count,
                                         const int64_t *counts, int counts_stride,
                                         int counts_first, int counts_n, int phase, int q_heads,
                                         int kv_heads, int head_dim, int page_size,
                                         void *workspace, size_t workspace_bytes,
                                         int32_t *device_status, hs_stream stream) {
  using namespace hs;
  if (int e = check_sizes(batch, dtype, pool_blocks, count, q_heads, kv_heads, head_dim,
                          page_size))
    return e;
  if (phase < 0 || phase > 1 || counts_n < 0 || counts_first < 0 || counts_stride < 0)
    return set_error(HS_ERR_INVALID_ARGUMENT, "attend_quantized: invalid phase or counts");
  if (batch == 0) return HS_OK;
  if (!query || (count > 0 && (!rows || !pool)))
    return set_error(HS_ERR_INVALID_ARGUMENT, "attend_quantized: null pointer");
  if ((reinterpret_cast<uintptr_t>(pool) & 15) != 0)
    return set_error(HS_ERR_INVALID_ARGUMENT,
                     "attend_quantized: the pool must be 16-byte aligned");
  QuantAttendParams p = params_of(batch, 2, dtype, q_heads, kv_heads, head_dim, count, workspace);
  if (int e = check_workspace(p, 2, workspace, workspace_bytes)) return e;
  p.query = query;
  p.q_batch_stride = query_batch_stride;
  p.pool = static_cast<const unsigned char *>(pool);
  p.pool_blocks = pool_blocks;
  p.rows = rows;
  p.rows_batch_stride = rows_batch_stride;
  p.counts64 = counts;
  p.counts_stride = counts_stride;
  p.counts_first = counts_first;
  p.counts_n = counts_n;
  p.phase = phase;
  p.page_size = page_size;
  p.page_shift = page_shift_of(page_size);
  p.status = device_status;
  return launch_rows(p, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int hs_attend_quantized_merge(int batch, int phases, void *out, int dtype, int q_heads,
                                         int kv_heads, int head_dim, int64_t count,
                                         void *workspace, size_t workspace_bytes,
                                         hs_stream stream) {
  using namespace hs;
  if (int e = check_sizes(batch, dtype, 0, count, q_heads, kv_heads, head_dim, 1)) return e;
  if (phases < 1 || phases > 2)
    return set_error(HS_ERR_INVALID_ARGUMENT, "attend_quantized: invalid number of phases");
  if (batch == 0) return HS_OK;
  if (!out) return set_error(HS_ERR_INVALID_ARGUMENT, "attend_quantized: null pointer");
  QuantAttendParams p = params_of(batch, 2, dtype, q_heads, kv_heads, head_dim, count, workspace);
  if (int e = check_workspace(p, 2, workspace, workspace_bytes)) return e;
  return launch_merge(p, phases, out, dtype, false, static_cast<cudaStream_t>(stream));
}
