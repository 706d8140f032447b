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
constexpr int kBwdRounds = 5;  // rounds of a backward block when there are rows enough

template <typename T> constexpr int unroll_of() { return sizeof(T) == 2 ? 4 : 2; }  // 64 bytes in flight a thread

// One row per cluster of blocks (one block when there are rows enough).  Each block finds the
// row's entries, marks the groups of eight columns that hold one in a bitmap, and runs once over
// its groups: a group without an entry goes to the running (maximum, sum) as it is; from the others
// the entries are taken out first (their logits go to the first block), so what is summed is the
// tail.  The first block joins the blocks' sums and one of its warps forms the loss.
template <typename T, bool SUM>
__global__ void __launch_bounds__(kFwdThreads) row_loss_fwd_kernel(const T* __restrict__ logits, int64_t ld,
                                                                   const int64_t* __restrict__ tids,
                                                                   const float* __restrict__ tlp, int K,
                                                                   RowLossParams P, RowState st,
                                                                   float* __restrict__ loss) {
  extern __shared__ uint32_t s_map[];  // a bit per group of this block
  __shared__ int s_col[kMaxEntries];
  __shared__ __align__(16) int s_raw[kMaxEntries];
  __shared__ float s_lp[kMaxEntries], s_x[kMaxEntries], s_red[64], s_part[3][8];
  constexpr int U = unroll_of<T>();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t r = blockIdx.x / C;
  const RowView<T> rv(logits, ld, r, P.V);
  const int per = (rv.groups + C - 1) / C;
  const int j0 = min(rank * per, rv.groups), j1 = min(j0 + per, rv.groups);

  int cnt = 0;
  const int64_t id = row_entries(tids + r * K, tlp ? tlp + r * K : nullptr, K, P.V, s_col, s_lp, s_raw, cnt);
  if (id == kRowLive) {
    for (int i = threadIdx.x; i < (per + 31) / 32; i += kFwdThreads) s_map[i] = 0u;
    __syncthreads();
    if (threadIdx.x < cnt) {
      const int j = (s_col[threadIdx.x] + rv.shift) >> 3;
      if (j >= j0 && j < j1) atomicOr(&s_map[(j - j0) >> 5], 1u << ((j - j0) & 31));
    }
    if (C > 1) cluster.sync();  // the first block's s_x and s_part exist before others write them
    else __syncthreads();
    float* x_dst = C > 1 ? cluster.map_shared_rank(s_x, 0) : s_x;

    float m = -INFINITY, s = 0.f, sum = 0.f;
    for (int jb = j0; jb < j1; jb += U * kFwdThreads) {
      Group8<T> g[U];
      const int n = min(U, (j1 - jb + kFwdThreads - 1) / kFwdThreads);  // groups a thread, at most
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jb + u * kFwdThreads + threadIdx.x;
        if (j < j1) load_group(g[u], rv, j);
        else g[u].fill();
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jb + u * kFwdThreads + threadIdx.x;
        if (j >= j1) continue;
        const int v0 = rv.first(j);
        if constexpr (SUM) {
          float x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = g[u].get(k);
          if (!rv.whole(j)) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (v0 + k < 0 || v0 + k >= P.V) x[k] = 0.f;
          }
          sum += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        }
        if ((s_map[(j - j0) >> 5] >> ((j - j0) & 31)) & 1u) {
          int lo = 0, hi = cnt;  // first entry at or after this group
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s_col[mid] < v0) lo = mid + 1;
            else hi = mid;
          }
          for (; lo < cnt && s_col[lo] < v0 + 8; ++lo) x_dst[lo] = g[u].take(s_col[lo] - v0);
        }
      }
      online_groups<T, U>(g, n, P.c, m, s);
    }
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
      part[8 + rank] = s;
      part[16 + rank] = sum;
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
  }
  if (rank != 0) return;
  if (threadIdx.x < K) st.cols[r * K + threadIdx.x] = s_col[threadIdx.x];
  if (threadIdx.x == 0) st.row_ids[r] = id;
  if (threadIdx.x < 32) {
    float m = -INFINITY, s = 0.f, sum = 0.f;
    if (id == kRowLive) {
      for (int q = 0; q < C; ++q) {
        online_merge(P.c, m, s, s_part[0][q], s_part[1][q]);
        sum += s_part[2][q];
      }
    }
    row_loss(P, id, cnt, s_x, s_lp, m, s, sum, loss + r, st.ref + r, st.coef + r, st.grad + r * K);
  }
}

// dlogits = g (coef 2^(c (x - ref)) + level) over the row, then g grad_k over its entries (written
// by the same block behind a barrier).  A block takes a part of one row, U groups a thread at a time;
// rows without a gradient are zeros and read nothing.
template <typename T>
__global__ void __launch_bounds__(kBwdThreads) row_loss_bwd_kernel(const T* __restrict__ logits, int64_t ld, int K,
                                                                   int V, float c, float level, RowState st,
                                                                   const float* __restrict__ dloss,
                                                                   T* __restrict__ dlogits, int64_t ld_out,
                                                                   int blocks_per_row) {
  constexpr int U = unroll_of<T>();
  const int64_t r = blockIdx.x / blocks_per_row;
  const int seg = (int)(blockIdx.x - r * blocks_per_row);
  const RowView<T> rv(logits, ld, r, V);
  T* out = dlogits + r * ld_out;
  const bool same = (reinterpret_cast<uintptr_t>(out) & 15) == (reinterpret_cast<uintptr_t>(rv.row) & 15);
  const int per = (rv.groups + blocks_per_row - 1) / blocks_per_row;
  const int j0 = min(seg * per, rv.groups), j1 = min(j0 + per, rv.groups);
  const float g = dloss[r], ref = st.ref[r], coef = st.coef[r];
  const bool skip = st.row_ids[r] == kRowNone || g == 0.f;
  const float lv = skip ? 0.f : g * level;
  // as in online_groups: one fma an exponent where c ref is finite, its rounding put into the factor
  const bool fma_ok = fabsf(ref) < kFmaLimit;
  const float pt = fma_ok ? ref * c : 0.f;
  const float gc = skip ? 0.f : g * coef * (fma_ok ? exp2f(-fmaf(ref, c, -pt)) : 1.f);

  for (int jb = j0; jb < j1; jb += U * kBwdThreads) {
    Group8<T> in[U];
    if (!skip) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jb + u * kBwdThreads + threadIdx.x;
        if (j < j1) load_group(in[u], rv, j);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = jb + u * kBwdThreads + threadIdx.x;
      if (j >= j1) break;
      float d[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (!skip) {
        if (fma_ok) {
#pragma unroll
          for (int k = 0; k < 8; ++k) d[k] = fmaf(gc, fast_exp2(fmaf(in[u].get(k), c, -pt)), lv);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) d[k] = fmaf(gc, fast_exp2((in[u].get(k) - ref) * c), lv);
        }
      }
      const int v0 = rv.first(j);
      if (same && rv.whole(j)) {
        if constexpr (sizeof(T) == 2) {
          st_stream16(out + v0, make_uint4(pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3]), pack_bf16x2(d[4], d[5]),
                                           pack_bf16x2(d[6], d[7])));
        } else {
          st_stream16(out + v0, make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]),
                                           __float_as_uint(d[3])));
          st_stream16(out + v0 + 4, make_uint4(__float_as_uint(d[4]), __float_as_uint(d[5]), __float_as_uint(d[6]),
                                               __float_as_uint(d[7])));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (v0 + k < 0 || v0 + k >= V) continue;
          if constexpr (sizeof(T) == 2) out[v0 + k] = f32_to_bf16_rn(d[k]);
          else out[v0 + k] = d[k];
        }
      }
    }
  }
  if (skip) return;
  __syncthreads();
  const int lo = rv.first(j0), hi = rv.first(j1);
  for (int e = threadIdx.x; e < K; e += kBwdThreads) {
    const int col = st.cols[r * K + e];
    if (col == kNoEntry || col < lo || col >= hi) continue;
    const float d = g * st.grad[r * K + e];
    if constexpr (sizeof(T) == 2) out[col] = f32_to_bf16_rn(d);
    else out[col] = d;
  }
}

// Entries of each row before the LM head's GEMM: one block a row.
__global__ void __launch_bounds__(kMaxEntries) row_entries_kernel(const int64_t* __restrict__ tids,
                                                                  const float* __restrict__ tlp, int K, int V,
                                                                  RowState st) {
  __shared__ int s_col[kMaxEntries];
  __shared__ __align__(16) int s_raw[kMaxEntries];
  __shared__ float s_lp[kMaxEntries];
  const int64_t r = blockIdx.x;
  int cnt = 0;
  const int64_t id = row_entries(tids + r * K, tlp ? tlp + r * K : nullptr, K, V, s_col, s_lp, s_raw, cnt);
  if (threadIdx.x < K) {
    st.cols[r * K + threadIdx.x] = s_col[threadIdx.x];
    st.grad[r * K + threadIdx.x] = s_lp[threadIdx.x];
  }
  if (threadIdx.x == 0) st.row_ids[r] = id;
}

// Loss of each row from partial sums: one warp a row.
__global__ void __launch_bounds__(128) row_losses_kernel(const float* __restrict__ part_m,
                                                         const float* __restrict__ part_s,
                                                         const float* __restrict__ part_x, int sets,
                                                         const int* __restrict__ pos, int64_t N, int K,
                                                         RowLossParams P, RowState st, float* __restrict__ loss,
                                                         const int* __restrict__ err) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= N) return;
  const int lane = threadIdx.x & 31;
  int64_t id = st.row_ids[r];
  if (err != nullptr && *err != 0) id = kRowBad;
  int cnt = 0;
  for (int k = lane; k < K; k += 32) cnt += st.cols[r * K + k] != kNoEntry;
  cnt = warp_sum(cnt);
  float m = -INFINITY, s = 0.f, sum = 0.f;
  if (id == kRowLive) {
    const int64_t at = pos ? pos[r] : r;
    for (int q = lane; q < sets; q += 32) {
      online_merge(P.c, m, s, part_m[(int64_t)q * N + at], part_s[(int64_t)q * N + at]);
      if (part_x) sum += part_x[(int64_t)q * N + at];
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    online_merge(P.c, m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  sum = warp_sum(sum);
  row_loss(P, id, cnt, st.xk + r * K, st.grad + r * K, m, s, sum, loss + r, st.ref + r, st.coef + r, st.grad + r * K);
}

template <typename T>
int launch_fwd(const void* logits, int64_t ld, const int64_t* tids, const float* tlp, int64_t N, int K,
               const RowLossParams& P, const RowState& st, float* loss, cudaStream_t s) {
  const int C = row_cluster(N, P.V, kFwdThreads);
  const int groups = (P.V + 7 + 7) / 8;
  const size_t smem = (size_t)(((groups + C - 1) / C + 31) / 32) * 4;
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
  const bool sum = P.loss == ROW_XENT && P.smoothing != 0.f;
  auto kern = sum ? row_loss_fwd_kernel<T, true> : row_loss_fwd_kernel<T, false>;
  IKRL_CUDA(cudaLaunchKernelEx(&cfg, kern, reinterpret_cast<const T*>(logits), ld, tids, tlp, K, P, st, loss));
  return check_launch("row_loss_fwd_kernel");
}

template <typename T>
int launch_bwd(const void* logits, int64_t ld, int64_t N, int K, int V, float c, float level, const RowState& st,
               const float* dloss, void* dlogits, int64_t ld_out, cudaStream_t s, const char* what) {
  const int groups = (V + 7 + 7) / 8;
  // Rows are cut so that a block runs a few rounds: its start (the row's scalars, then the first
  // loads) is paid once for them, while thousands of rows still even out over the SMs.
  const int per = unroll_of<T>() * kBwdThreads;
  const int rounds = N >= 8 * kNumSMs ? kBwdRounds : 1;
  const int bpr = (groups + per * rounds - 1) / (per * rounds);
  IKRL_REQUIRE(N * bpr <= 0x7fffffffLL, IKRL_ERR_UNSUPPORTED, "%s: N=%lld rows of V=%d need too many blocks", what,
               (long long)N, V);
  row_loss_bwd_kernel<T><<<(unsigned)(N * bpr), kBwdThreads, 0, s>>>(reinterpret_cast<const T*>(logits), ld, K, V, c,
                                                                     level, st, dloss, reinterpret_cast<T*>(dlogits),
                                                                     ld_out, bpr);
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
  *out = p;
  return IKRL_OK;
}

int launch_row_entries(const int64_t* tids, const float* tlp, int64_t N, int K, const RowLossParams& p,
                       const RowState& st, cudaStream_t s) {
  row_entries_kernel<<<(unsigned)N, kMaxEntries, 0, s>>>(tids, tlp, K, p.V, st);
  return check_launch("row_entries_kernel");
}

int launch_row_losses(const float* part_m, const float* part_s, const float* part_x, int sets, const int* pos,
                      int64_t N, int K, const RowLossParams& p, const RowState& st, float* loss, const int* err,
                      cudaStream_t s) {
  row_losses_kernel<<<(unsigned)((N + 3) / 4), 128, 0, s>>>(part_m, part_s, part_x, sets, pos, N, K, p, st, loss, err);
  return check_launch("row_losses_kernel");
}

}  // namespace ikrl

using namespace ikrl;

static int logits_loss_fwd(const char* what, const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V,
                           const int64_t* tids, const float* tlp, int32_t K, const RowLossParams& P, float* loss,
                           void* state, size_t state_bytes, void* stream) {
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
