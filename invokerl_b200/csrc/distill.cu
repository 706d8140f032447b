// Distillation and cross-entropy losses on logits in memory, forward and backward, and the row
// kernels that the LM head's forms of the same losses share (row_dist.cuh has the mathematics).
//
// Both directions are bound by HBM: the forward reads each logit once, the backward reads each
// once and writes its gradient once.
#include "row_dist.cuh"
#include "row_load.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace ikrl {
namespace {

namespace cg = cooperative_groups;

constexpr int kFwdThreads = 512;
constexpr int kBwdThreads = 512;
constexpr int kBwdRounds = 2;  // rounds of a backward block

template <typename T> constexpr int unroll_of() { return sizeof(T) == 2 ? 4 : 2; }  // 64 bytes in flight a thread

// Words of the bitmap of n groups, up to a whole round of the block.
__host__ __device__ __forceinline__ int map_words(int n) {
  return (n + kFwdThreads - 1) / kFwdThreads * (kFwdThreads / 32);
}

// A row's entries in a forward block: their columns ascending, a bit for each whole group of the part
// that holds one (bit j - a), and where their logits go.
struct RowEntries {
  const int* col;
  int cnt;
  const uint32_t* map;
  float* x;
};

template <typename T>
__device__ __forceinline__ void mark_entry(const RowPart<T>& p, int col, uint32_t* map) {
  const int j = p.group_of(col);
  if (j >= p.a && j < p.b) atomicOr(&map[(j - p.a) >> 5], 1u << ((j - p.a) & 31));
}

// U groups a thread of a part from group jb on; behind the part's last, groups of -inf.
template <typename T, int U>
__device__ __forceinline__ void load_round(Group8<T> (&g)[U], const RowPart<T>& p, int jb) {
  if (jb + U * kFwdThreads <= p.b) {
#pragma unroll
    for (int u = 0; u < U; ++u) g[u].load(p.at(jb + u * kFwdThreads + (int)threadIdx.x));
    return;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int j = jb + u * kFwdThreads + (int)threadIdx.x;
    if (j < p.b) g[u].load(p.at(j));
    else g[u].fill();
  }
}

// Sum of a group in units of kSumUnit.
template <typename T>
__device__ __forceinline__ float group_sum(const Group8<T>& g) {
  const uint64_t u = pack2(1.f / kSumUnit, 1.f / kSumUnit);
  float lo, hi;
  unpack2(add2(fma2(g.get2(1), u, mul2(g.get2(0), u)), fma2(g.get2(3), u, mul2(g.get2(2), u))), lo, hi);
  return lo + hi;
}

// Running sums of a part by a block: m, s over the tail and, with SUM, the sum of all logits (in kSumUnit).
//
// The loop over the part leaves out the groups that hold entries: their bits are one shared word a
// warp and group, zero most of the time.  Those groups are taken one a thread, by the thread of their
// first entry, and so are the groups that reach past the row.  g holds the first round.
template <typename T, int U, bool SUM>
__device__ __forceinline__ void sum_part(Group8<T> (&g)[U], const RowPart<T>& p, const RowEntries& e, float c, float& m,
                                         float& s, float& sum) {
  const int tid = (int)threadIdx.x;
  int mine = -1, first = 0;
  if (tid < e.cnt) {
    const int j = p.group_of(e.col[tid]);
    if (j >= p.j0 && j < p.j1 && (tid == 0 || p.group_of(e.col[tid - 1]) != j)) {
      mine = j;
      first = tid;
    }
  }
  // The block's last two threads take the edges that hold no entry.
  const int ej = p.edge(kFwdThreads - 1 - tid);
  if (ej >= 0) {
    bool holds = false;
    for (int k = 0; k < e.cnt; ++k) holds |= p.group_of(e.col[k]) == ej;
    if (!holds) {
      mine = ej;
      first = e.cnt;
    }
  }
  if (mine >= 0) {
    Group8<T> h[1];
    load_group(h[0], p.rv, mine);
    const int v0 = p.rv.first(mine);
    if constexpr (SUM) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (v0 + k >= 0 && v0 + k < p.rv.V) sum = fmaf(h[0].get(k), 1.f / kSumUnit, sum);
    }
    for (; first < e.cnt && e.col[first] < v0 + 8; ++first) e.x[first] = h[0].take(e.col[first] - v0);
    online_groups<T, 1>(h, c, m, s);
  }

  int jb = p.a;
  const uint32_t* word = e.map + (tid >> 5);
  const uint32_t bit = 1u << (tid & 31);
  for (; jb + U * kFwdThreads <= p.b; jb += U * kFwdThreads) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t wd = word[u * (kFwdThreads / 32)];
      if constexpr (SUM) {
        const float x = group_sum(g[u]);
        sum += (wd & bit) ? 0.f : x;
      }
      if (wd != 0 && (wd & bit)) g[u].fill();
    }
    word += U * (kFwdThreads / 32);
    online_groups<T, U>(g, c, m, s);
    if (jb + U * kFwdThreads < p.b) load_round<T, U>(g, p, jb + U * kFwdThreads);
  }
  if (jb < p.b) {  // the last round, in part
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = jb + u * kFwdThreads + tid < p.b;
      const bool entry = jb + u * kFwdThreads < p.b && (word[u * (kFwdThreads / 32)] & bit);  // the map ends with p.b
      if constexpr (SUM) {
        if (in && !entry) sum += group_sum(g[u]);
      }
      if (entry) g[u].fill();
    }
    online_groups<T, U>(g, c, m, s);
  }
}

// Few rows: one launch.  A cluster of blocks shares a row (one block when it is short); each finds the
// row's entries and sums its part, the first block joins the parts and one of its warps forms the loss.
template <typename T, bool SUM>
__global__ void __launch_bounds__(kFwdThreads) row_loss_fwd_kernel(const T* __restrict__ logits, int64_t ld,
                                                                   const int64_t* __restrict__ tids,
                                                                   const float* __restrict__ tlp, int K,
                                                                   RowLossParams P, RowState st,
                                                                   float* __restrict__ loss) {
  extern __shared__ uint32_t s_map[];
  __shared__ int s_col[kMaxEntries];
  __shared__ int s_raw[kMaxEntries];
  __shared__ float s_lp[kMaxEntries], s_x[kMaxEntries], s_red[64], s_part[3][kMaxParts];
  constexpr int U = unroll_of<T>();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t r = blockIdx.x / C;
  const RowPart<T> p(logits, ld, r, P.V, rank, C);
  Group8<T> g[U];
  load_round<T, U>(g, p, p.a);

  for (int i = threadIdx.x; i < map_words(p.b - p.a); i += kFwdThreads) s_map[i] = 0u;
  int cnt = 0;
  const int64_t id = row_entries(tids + r * K, tlp ? tlp + r * K : nullptr, K, P.V, s_col, s_lp, s_raw, cnt);
  if (threadIdx.x < cnt) mark_entry(p, s_col[threadIdx.x], s_map);
  if (C > 1) cluster.sync();  // the first block's s_x and s_part exist before others write them
  else __syncthreads();
  const RowEntries e{s_col, cnt, s_map, C > 1 ? cluster.map_shared_rank(s_x, 0) : s_x};

  float m = -INFINITY, s = 0.f, sum = 0.f;
  sum_part<T, U, SUM>(g, p, e, P.c, m, s, sum);
  block_online_merge(P.c, m, s, s_red);
  if constexpr (SUM) {
    float v[1] = {sum};
    __syncthreads();
    block_sum<float, 1>(v, s_red);
    sum = v[0];
  }
  if (threadIdx.x == 0) {
    float* part = C > 1 ? cluster.map_shared_rank(&s_part[0][0], 0) : &s_part[0][0];
    part[rank] = m;
    part[kMaxParts + rank] = s;
    part[2 * kMaxParts + rank] = sum;
  }
  if (C > 1) cluster.sync();
  else __syncthreads();
  if (rank != 0) return;
  if (threadIdx.x < K) st.cols[r * K + threadIdx.x] = s_col[threadIdx.x];
  if (threadIdx.x == 0) st.row_ids[r] = id;
  if (threadIdx.x < 32) {
    m = -INFINITY;
    s = sum = 0.f;
    for (int q = 0; q < C; ++q) {
      online_merge(P.c, m, s, s_part[0][q], s_part[1][q]);
      sum += s_part[2][q];
    }
    row_loss(P, id, cnt, s_x, s_lp, m, s, sum, loss + r, st.ref + r, st.coef + r, st.grad + r * K);
  }
}

// Many rows: the sums between row_entries_kernel and row_losses_kernel, one block a part of a row.
// Rows without entries are not read.
template <typename T, bool SUM, int U, int MINB>
__global__ void __launch_bounds__(kFwdThreads, MINB) row_sums_kernel(const T* __restrict__ logits, int64_t ld,
                                                                     RowCut cut, int K, float c, int V, RowState st,
                                                                     int64_t N) {
  extern __shared__ uint32_t s_map[];
  __shared__ int s_cols[kMaxEntries];
  __shared__ float s_red[64], s_sum[32];
  int64_t r = blockIdx.x;
  int seg = 0, segs = 1;
  if (r >= cut.whole) {
    const unsigned b = (unsigned)(r - cut.whole);
    segs = cut.parts;  // a power of two
    r = cut.whole + (b >> (31 - __clz(segs)));
    seg = (int)(b & (unsigned)(segs - 1));
  }
  const RowPart<T> p(logits, ld, r, V, seg, segs);
  Group8<T> g[U];
  load_round<T, U>(g, p, p.a);  // a row that is not live costs this read
  const int64_t id = st.row_ids[r];
  const int col = threadIdx.x < K ? st.cols[r * K + threadIdx.x] : kNoEntry;
  for (int i = threadIdx.x; i < map_words(p.b - p.a); i += kFwdThreads) s_map[i] = 0u;
  if (threadIdx.x < K) s_cols[threadIdx.x] = col;
  if (id != kRowLive) return;
  __syncthreads();
  if (col != kNoEntry) mark_entry(p, col, s_map);
  const int cnt = __syncthreads_count(col != kNoEntry);
  float m = -INFINITY, s = 0.f, sum = 0.f;
  sum_part<T, U, SUM>(g, p, RowEntries{s_cols, cnt, s_map, st.xk + r * K}, c, m, s, sum);
  if constexpr (SUM) {
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
  }
  block_online_merge(c, m, s, s_red);
  if (threadIdx.x < 32) {
    if constexpr (SUM) sum = warp_sum(threadIdx.x < kFwdThreads / 32 ? s_sum[threadIdx.x] : 0.f);
    if (threadIdx.x == 0) {
      st.part[(int64_t)seg * N + r] = m;
      st.part[((int64_t)kMaxParts + seg) * N + r] = s;
      if constexpr (SUM) st.part[((int64_t)2 * kMaxParts + seg) * N + r] = sum;
    }
    if (segs < cut.parts && threadIdx.x > 0 && threadIdx.x < cut.parts) {  // the parts that a whole row lacks
      st.part[(int64_t)threadIdx.x * N + r] = -INFINITY;
      st.part[((int64_t)kMaxParts + threadIdx.x) * N + r] = 0.f;
      if constexpr (SUM) st.part[((int64_t)2 * kMaxParts + threadIdx.x) * N + r] = 0.f;
    }
  }
}

// One group of the gradient.
template <typename T>
__device__ __forceinline__ void store_group(T* __restrict__ out, const float (&d)[8]) {
  if constexpr (sizeof(T) == 2) {
    st_stream16(out, make_uint4(pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3]), pack_bf16x2(d[4], d[5]),
                                pack_bf16x2(d[6], d[7])));
  } else {
    st_stream16(out, make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]),
                                __float_as_uint(d[3])));
    st_stream16(out + 4, make_uint4(__float_as_uint(d[4]), __float_as_uint(d[5]), __float_as_uint(d[6]),
                                    __float_as_uint(d[7])));
  }
}
template <typename T>
__device__ __forceinline__ void store_value(T* out, float d) {
  if constexpr (sizeof(T) == 2) *out = f32_to_bf16_rn(d);
  else *out = d;
}

// dlogits = g (coef 2^(c (x - ref)) + level) over the row, then g grad_k over its entries (written
// by the same block behind a barrier).  One block a part of a row; rows without a gradient are zeros
// and read nothing.
template <typename T, int U, int MINB>
__global__ void __launch_bounds__(kBwdThreads, MINB) row_loss_bwd_kernel(const T* __restrict__ logits, int64_t ld,
                                                                         int K, int V, float c, float level,
                                                                         RowState st, const float* __restrict__ dloss,
                                                                         T* __restrict__ dlogits, int64_t ld_out,
                                                                         int segs) {
  const int64_t r = blockIdx.x / segs;
  const int seg = (int)(blockIdx.x - r * segs);
  const RowPart<T> p(logits, ld, r, V, seg, segs);
  T* out = dlogits + r * ld_out;
  const float g = dloss[r], ref = st.ref[r], coef = st.coef[r];
  const bool skip = st.row_ids[r] == kRowNone || g == 0.f;
  const bool same = (reinterpret_cast<uintptr_t>(out) & 15) == (reinterpret_cast<uintptr_t>(p.rv.row) & 15);
  if (skip && same) {
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j = p.a + (int)threadIdx.x; j < p.b; j += kBwdThreads) store_group<T>(out + p.rv.first(j), zero);
    const int j = p.edge(threadIdx.x);
    if (j >= 0)
      for (int v = max(p.rv.first(j), 0); v < min(p.rv.first(j) + 8, V); ++v) store_value<T>(out + v, 0.f);
    return;
  }
  const float lv = skip ? 0.f : g * level;
  // as in online_groups: one fma an exponent where c ref is small enough, its rounding put into the factor
  const float pt = ref * c;
  const bool fma_ok = fabsf(pt) < kFmaLimit;
  const float gc = skip ? 0.f : g * coef * (fma_ok ? exp2f(-fmaf(ref, c, -pt)) : 1.f);
  if (fma_ok && same) {
    const uint64_t c2 = pack2(c, c), npt2 = pack2(-pt, -pt), gc2 = pack2(gc, gc), lv2 = pack2(lv, lv);
    for (int jb = p.a; jb < p.b; jb += U * kBwdThreads) {
      Group8<T> in[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jb + u * kBwdThreads + (int)threadIdx.x;
        if (j < p.b) in[u].load(p.rv.row + p.rv.first(j));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jb + u * kBwdThreads + (int)threadIdx.x;
        if (j >= p.b) break;
        float d[8];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          unpack2(fma2(gc2, exp2x2(fma2(in[u].get2(k), c2, npt2)), lv2), d[2 * k], d[2 * k + 1]);
        store_group<T>(out + p.rv.first(j), d);
      }
    }
    const int j = p.edge(threadIdx.x);
    if (j >= 0) {
      Group8<T> e;
      load_group(e, p.rv, j);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int v = p.rv.first(j) + k;
        if (v >= 0 && v < V) store_value<T>(out + v, fmaf(gc, fast_exp2(fmaf(e.get(k), c, -pt)), lv));
      }
    }
  } else {
    // outputs placed unlike the inputs, or a tail that holds nothing or nothing but masks
    const int lo = max(p.rv.first(p.j0), 0), hi = min(p.rv.first(p.j1), V);
    for (int v = lo + (int)threadIdx.x; v < hi; v += kBwdThreads) {
      float d = 0.f;
      if (!skip) {
        float x;
        if constexpr (sizeof(T) == 2) x = bf16_to_f32(p.rv.row[v]);
        else x = p.rv.row[v];
        d = fmaf(g * coef, fast_exp2((x - ref) * c), lv);
      }
      store_value<T>(out + v, d);
    }
  }
  if (skip) return;
  __syncthreads();
  const int lo = p.rv.first(p.j0), hi = p.rv.first(p.j1);
  for (int e = threadIdx.x; e < K; e += kBwdThreads) {
    const int col = st.cols[r * K + e];
    if (col == kNoEntry || col < lo || col >= hi) continue;
    store_value<T>(out + col, g * st.grad[r * K + e]);
  }
}

// Entries of each row: one block a row, or one thread for a single target.
__global__ void row_entries_kernel(const int64_t* __restrict__ tids, const float* __restrict__ tlp, int K, int V,
                                   RowState st, int* __restrict__ clear) {
  __shared__ int s_col[kMaxEntries];
  __shared__ int s_raw[kMaxEntries];
  __shared__ float s_lp[kMaxEntries];
  const int64_t r = blockIdx.x;
  int cnt = 0;
  const int64_t id = row_entries(tids + r * K, tlp + r * K, K, V, s_col, s_lp, s_raw, cnt);
  if (threadIdx.x < K) {
    st.cols[r * K + threadIdx.x] = s_col[threadIdx.x];
    st.grad[r * K + threadIdx.x] = s_lp[threadIdx.x];
  }
  if (threadIdx.x == 0) st.row_ids[r] = id;
  if (r == 0 && threadIdx.x == 0 && clear != nullptr) *clear = 0;
}

__global__ void row_targets_kernel(const int64_t* __restrict__ targets, int64_t N, int V, RowState st,
                                   int* __restrict__ clear) {
  const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (r == 0 && clear != nullptr) *clear = 0;
  if (r >= N) return;
  const int64_t t = targets[r];
  const bool ok = t >= 0 && t < V;
  st.cols[r] = ok ? (int)t : kNoEntry;
  st.row_ids[r] = ok ? kRowLive : (t == -100 ? kRowNone : kRowBad);
}

// Loss of each row from partial sums: WARPS warps a row (they share its partial sums; the first forms the
// loss), four warps a block.
template <int WARPS>
__global__ void __launch_bounds__(128) row_losses_kernel(const float* __restrict__ part_m,
                                                         const float* __restrict__ part_s,
                                                         const float* __restrict__ part_x, int sets,
                                                         const int* __restrict__ sets_dev,
                                                         const int* __restrict__ pos, int64_t N, int K,
                                                         RowLossParams P, RowState st, float* __restrict__ loss,
                                                         const int* __restrict__ err) {
  static_assert(WARPS == 1 || WARPS == 4, "a block's four warps take four rows or one");
  __shared__ float s_part[3][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (4 / WARPS) + (WARPS == 1 ? warp : 0);
  if (r >= N) return;
  int64_t id = st.row_ids[r];
  if (err != nullptr && *err != 0) id = kRowBad;
  float m = -INFINITY, s = 0.f, sum = 0.f;
  if (id == kRowLive) {
    const int64_t at = pos ? pos[r] : r;
    if (sets_dev != nullptr) sets = *sets_dev;
    for (int q = WARPS == 1 ? lane : (int)threadIdx.x; q < sets; q += 32 * WARPS) {
      online_merge(P.c, m, s, part_m[(int64_t)q * N + at], part_s[(int64_t)q * N + at]);
      if (part_x) sum += part_x[(int64_t)q * N + at];
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    online_merge(P.c, m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  sum = warp_sum(sum);
  if constexpr (WARPS == 4) {
    if (lane == 0) {
      s_part[0][warp] = m;
      s_part[1][warp] = s;
      s_part[2][warp] = sum;
    }
    __syncthreads();
    if (warp != 0) return;
    m = -INFINITY;
    s = sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      online_merge(P.c, m, s, s_part[0][w], s_part[1][w]);
      sum += s_part[2][w];
    }
  }
  int cnt = 0;
  for (int k = lane; k < K; k += 32) cnt += st.cols[r * K + k] != kNoEntry;
  cnt = warp_sum(cnt);
  row_loss(P, id, cnt, st.xk + r * K, st.grad + r * K, m, s, sum, loss + r, st.ref + r, st.coef + r, st.grad + r * K);
}

// Rows up to which a forward is one launch with clusters sharing rows, all blocks at once; above, three
// launches.  Distillation forward, 64 entries of 151936 bf16 columns, 64 / 148 / 296 rows: 18 / 23 / 30 us in one
// launch, 28 / 32 / 40 us in three.
constexpr int64_t kFusedRows = 2 * kNumSMs;

template <typename T>
int launch_fwd(const void* logits, int64_t ld, const int64_t* tids, const float* tlp, int64_t N, int K,
               const RowLossParams& P, const RowState& st, float* loss, cudaStream_t s) {
  const bool sum = P.loss == ROW_XENT && P.smoothing != 0.f;
  const int groups = (P.V + 7 + 7) / 8;
  const T* x = reinterpret_cast<const T*>(logits);
  if (N <= kFusedRows) {
    const int C = row_cluster(N, P.V, kFwdThreads);
    const size_t smem = (size_t)map_words((groups + C - 1) / C) * 4;
    auto kern = sum ? row_loss_fwd_kernel<T, true> : row_loss_fwd_kernel<T, false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(N * C), 1, 1);
    cfg.blockDim = dim3(kFwdThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    IKRL_CUDA(cudaLaunchKernelEx(&cfg, kern, x, ld, tids, tlp, K, P, st, loss));
    return check_launch("row_loss_fwd_kernel");
  }
  int rc = launch_row_entries(tids, tlp, N, K, P, st, s);
  if (rc) return rc;
  constexpr int U = unroll_of<T>();
  static_assert(kMaxRowParts <= kMaxParts, "the state holds a sum for every part");
  const RowCut cut = row_cut(N, P.V, sizeof(T), kFwdThreads * U);
  const int64_t blocks = cut.whole + (N - cut.whole) * cut.parts;
  IKRL_REQUIRE(blocks <= 0x7fffffffLL, IKRL_ERR_UNSUPPORTED, "N=%lld rows of V=%d need too many blocks",
               (long long)N, P.V);
  const size_t smem = (size_t)map_words(cut.whole > 0 ? groups : (groups + cut.parts - 1) / cut.parts) * 4;
  auto kern = sum ? row_sums_kernel<T, true, U, 4> : row_sums_kernel<T, false, U, 4>;
  kern<<<(unsigned)blocks, kFwdThreads, smem, s>>>(x, ld, cut, K, P.c, P.V, st, N);
  if ((rc = check_launch("row_sums_kernel"))) return rc;
  const float* part = st.part;
  return launch_row_losses(part, part + (int64_t)kMaxParts * N, sum ? part + (int64_t)2 * kMaxParts * N : nullptr,
                           cut.parts, nullptr, nullptr, N, K, P, st, loss, nullptr, s);
}

template <typename T>
int launch_bwd(const void* logits, int64_t ld, int64_t N, int K, int V, float c, float level, const RowState& st,
               const float* dloss, void* dlogits, int64_t ld_out, cudaStream_t s, const char* what) {
  const int groups = (V + 7 + 7) / 8;
  constexpr int U = unroll_of<T>();
  const int segs = std::max(1, groups / (kBwdThreads * U * kBwdRounds));
  IKRL_REQUIRE(N * segs <= 0x7fffffffLL, IKRL_ERR_UNSUPPORTED, "%s: N=%lld rows of V=%d need too many blocks", what,
               (long long)N, V);
  row_loss_bwd_kernel<T, U, 3><<<(unsigned)(N * segs), kBwdThreads, 0, s>>>(
      reinterpret_cast<const T*>(logits), ld, K, V, c, level, st, dloss, reinterpret_cast<T*>(dlogits), ld_out, segs);
  return check_launch("row_loss_bwd_kernel");
}

int check_state(const char* what, const void* state, size_t state_bytes, int64_t N, int K) {
  const size_t need = row_state_bytes(N, K);
  IKRL_REQUIRE(state != nullptr && state_bytes >= need, IKRL_ERR_WORKSPACE, "%s: state %zu < %zu bytes", what,
               state_bytes, need);
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(state) & 255) == 0, IKRL_ERR_ALIGNMENT,
               "%s: state must be 256-byte aligned", what);
  return IKRL_OK;
}

}  // namespace

int check_logits_arg(const char* what, const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V) {
  IKRL_REQUIRE(N >= 0 && V > 0 && ld >= V, IKRL_ERR_INVALID_ARGUMENT, "%s: bad sizes N=%lld V=%d ld=%lld", what,
               (long long)N, V, (long long)ld);
  IKRL_REQUIRE(dtype == IKRL_DTYPE_F32 || dtype == IKRL_DTYPE_BF16, IKRL_ERR_UNSUPPORTED, "%s: dtype %d unsupported",
               what, dtype);
  IKRL_REQUIRE(V <= kMaxVocab, IKRL_ERR_UNSUPPORTED, "%s: V=%d exceeds %d columns", what, V, kMaxVocab);
  IKRL_REQUIRE(N <= (0x7fffffffLL / 8), IKRL_ERR_UNSUPPORTED, "%s: N=%lld too large", what, (long long)N);
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype == IKRL_DTYPE_F32 ? 3 : 1)) == 0, IKRL_ERR_ALIGNMENT,
               "%s: logits must be aligned to their type", what);
  return IKRL_OK;
}

int distill_params(const char* what, const ikrl_distill_params* d, int V, int K, RowLossParams* out) {
  IKRL_REQUIRE(d != nullptr, IKRL_ERR_INVALID_ARGUMENT, "%s: params is NULL", what);
  IKRL_REQUIRE(d->kind >= IKRL_DISTILL_FORWARD && d->kind <= IKRL_DISTILL_JSD, IKRL_ERR_INVALID_ARGUMENT,
               "%s: kind %d not in 0..2", what, d->kind);
  IKRL_REQUIRE(d->temperature > 0.f && isfinite(d->temperature), IKRL_ERR_INVALID_ARGUMENT,
               "%s: temperature %g must be positive and finite", what, (double)d->temperature);
  IKRL_REQUIRE(d->tail || d->kind == IKRL_DISTILL_FORWARD, IKRL_ERR_UNSUPPORTED,
               "%s: the reverse and JSD losses need the tail outcome", what);
  IKRL_REQUIRE(d->kind != IKRL_DISTILL_JSD || (d->beta > 0.f && d->beta < 1.f), IKRL_ERR_INVALID_ARGUMENT,
               "%s: beta %g outside (0, 1)", what, (double)d->beta);
  IKRL_REQUIRE(K >= 1 && K <= kMaxEntries, IKRL_ERR_UNSUPPORTED, "%s: K=%d entries outside 1..%d", what, K,
               kMaxEntries);
  IKRL_REQUIRE(V < 1 << 24, IKRL_ERR_UNSUPPORTED, "%s: V=%d needs more than 24 bits", what, V);  // row_entries
  RowLossParams p{};
  p.loss = d->kind == IKRL_DISTILL_FORWARD ? (d->tail ? ROW_FORWARD : ROW_FORWARD_TOPK)
                                           : (d->kind == IKRL_DISTILL_REVERSE ? ROW_REVERSE : ROW_JSD);
  p.V = V;
  p.c = (float)(1.4426950408889634 / (double)d->temperature);
  p.inv_t = (float)(1.0 / (double)d->temperature);
  p.beta = d->beta;
  IKRL_REQUIRE(p.c > 0.f && isfinite(p.c), IKRL_ERR_INVALID_ARGUMENT, "%s: temperature %g out of range", what,
               (double)d->temperature);
  *out = p;
  return IKRL_OK;
}

int xent_params(const char* what, float smoothing, float z_loss, int V, RowLossParams* out) {
  IKRL_REQUIRE(smoothing >= 0.f && smoothing <= 1.f, IKRL_ERR_INVALID_ARGUMENT,
               "%s: label smoothing %g outside [0, 1]", what, (double)smoothing);
  IKRL_REQUIRE(isfinite(z_loss), IKRL_ERR_INVALID_ARGUMENT, "%s: z_loss %g is not finite", what, (double)z_loss);
  RowLossParams p{};
  p.loss = ROW_XENT;
  p.V = V;
  p.c = kLog2e;
  p.inv_t = 1.f;
  p.smoothing = smoothing;
  p.zeta = z_loss;
  p.sum_unit = 1.f;
  *out = p;
  return IKRL_OK;
}

int launch_row_entries(const int64_t* tids, const float* tlp, int64_t N, int K, const RowLossParams& p,
                       const RowState& st, cudaStream_t s, int* clear) {
  if (tlp == nullptr) {
    row_targets_kernel<<<(unsigned)((N + 255) / 256), 256, 0, s>>>(tids, N, p.V, st, clear);
    return check_launch("row_targets_kernel");
  }
  row_entries_kernel<<<(unsigned)N, (unsigned)entry_threads(K), 0, s>>>(tids, tlp, K, p.V, st, clear);
  return check_launch("row_entries_kernel");
}

int launch_row_losses(const float* part_m, const float* part_s, const float* part_x, int sets,
                      const int* sets_dev, const int* pos, int64_t N, int K, const RowLossParams& p, const RowState& st,
                      float* loss, const int* err, cudaStream_t s) {
  if (row_takes_a_block(sets, N))
    row_losses_kernel<4><<<(unsigned)N, 128, 0, s>>>(part_m, part_s, part_x, sets, sets_dev, pos, N, K, p, st, loss,
                                                        err);
  else
    row_losses_kernel<1><<<(unsigned)((N + 3) / 4), 128, 0, s>>>(part_m, part_s, part_x, sets, sets_dev, pos, N, K,
                                                                 p, st, loss, err);
  return check_launch("row_losses_kernel");
}

}  // namespace ikrl

using namespace ikrl;

static int logits_loss_fwd(const char* what, const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V,
                           const int64_t* tids, const float* tlp, int32_t K, RowLossParams P, float* loss,
                           void* state, size_t state_bytes, void* stream) {
  P.sum_unit = kSumUnit;
  int rc = check_logits_arg(what, logits, dtype, ld, N, V);
  if (rc || N == 0) return rc;
  IKRL_REQUIRE(logits && tids && loss, IKRL_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if ((rc = check_state(what, state, state_bytes, N, K))) return rc;
  const RowState st = row_state(state, N, K);
  return dtype == IKRL_DTYPE_BF16
             ? launch_fwd<uint16_t>(logits, ld, tids, tlp, N, K, P, st, loss, as_stream(stream))
             : launch_fwd<float>(logits, ld, tids, tlp, N, K, P, st, loss, as_stream(stream));
}

static int logits_loss_bwd(const char* what, const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V,
                           int32_t K, const RowLossParams& P, const void* state, size_t state_bytes,
                           const float* dloss, void* dlogits, int64_t ld_out, void* stream) {
  int rc = check_logits_arg(what, logits, dtype, ld, N, V);
  if (rc || N == 0) return rc;
  IKRL_REQUIRE(ld_out >= V, IKRL_ERR_INVALID_ARGUMENT, "%s: ld_out=%lld < V=%d", what, (long long)ld_out, V);
  IKRL_REQUIRE(logits && dloss && dlogits, IKRL_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(dlogits) & (dtype == IKRL_DTYPE_F32 ? 3 : 1)) == 0, IKRL_ERR_ALIGNMENT,
               "%s: dlogits must be aligned to their type", what);
  if ((rc = check_state(what, state, state_bytes, N, K))) return rc;
  const RowState st = row_state(const_cast<void*>(state), N, K);
  const float level = P.loss == ROW_XENT ? -P.smoothing / (float)V : 0.f;
  return dtype == IKRL_DTYPE_BF16 ? launch_bwd<uint16_t>(logits, ld, N, K, V, P.c, level, st, dloss, dlogits, ld_out,
                                                         as_stream(stream), what)
                                  : launch_bwd<float>(logits, ld, N, K, V, P.c, level, st, dloss, dlogits, ld_out,
                                                      as_stream(stream), what);
}

extern "C" {

size_t ikrl_row_loss_state_bytes(int64_t N, int32_t K) {
  if (N <= 0 || K <= 0) return 256;
  return row_state_bytes(N, K);
}

int ikrl_logits_distill_fwd(const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V,
                            const int64_t* teacher_ids, const float* teacher_logp, int32_t K,
                            const ikrl_distill_params* params, float* loss, void* state, size_t state_bytes,
                            void* stream) {
  clear_error();
  const char* what = "ikrl_logits_distill_fwd";
  RowLossParams P;
  int rc = distill_params(what, params, V, K, &P);
  if (rc) return rc;
  IKRL_REQUIRE(N <= 0 || teacher_logp, IKRL_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  return logits_loss_fwd(what, logits, dtype, ld, N, V, teacher_ids, teacher_logp, K, P, loss, state, state_bytes,
                         stream);
}

int ikrl_logits_distill_bwd(const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V, int32_t K,
                            const ikrl_distill_params* params, const void* state, size_t state_bytes,
                            const float* dloss, void* dlogits, int64_t ld_out, void* stream) {
  clear_error();
  const char* what = "ikrl_logits_distill_bwd";
  RowLossParams P;
  int rc = distill_params(what, params, V, K, &P);
  if (rc) return rc;
  return logits_loss_bwd(what, logits, dtype, ld, N, V, K, P, state, state_bytes, dloss, dlogits, ld_out, stream);
}

int ikrl_logits_cross_entropy_fwd(const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V,
                                  const int64_t* targets, float label_smoothing, float z_loss, float* loss,
                                  void* state, size_t state_bytes, void* stream) {
  clear_error();
  const char* what = "ikrl_logits_cross_entropy_fwd";
  RowLossParams P;
  int rc = xent_params(what, label_smoothing, z_loss, V, &P);
  if (rc) return rc;
  return logits_loss_fwd(what, logits, dtype, ld, N, V, targets, nullptr, 1, P, loss, state, state_bytes, stream);
}

int ikrl_logits_cross_entropy_bwd(const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V,
                                  float label_smoothing, float z_loss, const void* state, size_t state_bytes,
                                  const float* dloss, void* dlogits, int64_t ld_out, void* stream) {
  clear_error();
  const char* what = "ikrl_logits_cross_entropy_bwd";
  RowLossParams P;
  int rc = xent_params(what, label_smoothing, z_loss, V, &P);
  if (rc) return rc;
  return logits_loss_bwd(what, logits, dtype, ld, N, V, 1, P, state, state_bytes, dloss, dlogits, ld_out, stream);
}

}  // extern "C"
