// The k likeliest tokens of each row of logits and their log-probs over the whole vocabulary: what
// a teacher gives a distillation.
//
// One pass over the row, bound by HBM.  Beside the running logsumexp, a block notes the groups of
// eight columns whose maximum reaches a bar, a lower bound of the k-th largest value: the k-th largest
// of the threads' own maxima so far, found bit by bit with block-wide counts and raised after 1, 2,
// 4, 8, ... rounds.  With 512 threads that bound is nearly the k-th largest itself, so of V columns in
// no particular order about k (1 + log2(V / 16384)) are noted.  The noted groups are read again (from
// L2), their columns above the bar go to a buffer of keys, and the buffer is sorted.  Where a list
// fills up (rising rows, many equal values) it is worked off, and the keys are cut to the k largest,
// which raises the bar to the k-th key itself.
//
// Order and ties are those of one 64-bit key, the value above the inverted column: larger values
// first, of equal values the lower column.  Keys are distinct, so the result does not depend on the
// order in which columns enter.
#include "row_dist.cuh"
#include "row_load.cuh"

#include <cooperative_groups.h>

namespace ikrl {
namespace {

namespace cg = cooperative_groups;

constexpr int kTopThreads = 512;
constexpr int kTopBuf = 2048;  // keys of the buffer: the cluster's 8 x kMaxEntries at the end
constexpr int kTopList = 4096;  // noted groups
static_assert(kTopBuf >= 8 * kMaxEntries && kTopBuf >= 2 * kMaxEntries, "top-k buffer too small");

// Values in key order: NaN first, -0 as +0.
__device__ __forceinline__ uint32_t value_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return nan_f32();
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// Sort s[0, n) descending, n a power of two; the keys behind `have` count as 0.  Bitonic: up to one key a
// thread, the exchanges inside a warp are shuffles and only those between warps go through memory.
__device__ __forceinline__ void sort_keys(uint64_t* s, int have, int n) {
  const int t = (int)threadIdx.x;
  if (n <= kTopThreads) {
    uint64_t x = t < have ? s[t] : 0;
    for (int k = 2; k <= n; k <<= 1) {
      const bool down = (t & k) == 0;
      int j = k >> 1;
      for (; j >= 32; j >>= 1) {
        __syncthreads();
        if (t < n) s[t] = x;
        __syncthreads();
        if (t < n) {
          const uint64_t y = s[t ^ j];
          if (((t & j) == 0) == down ? x < y : x > y) x = y;
        }
      }
      if ((t & ~31) < n) {  // whole warps
        for (; j > 0; j >>= 1) {
          const uint64_t y = __shfl_xor_sync(0xffffffffu, x, j);
          if (((t & j) == 0) == down ? x < y : x > y) x = y;
        }
      }
    }
    __syncthreads();
    if (t < n) s[t] = x;
    __syncthreads();
    return;
  }
  for (int i = have + t; i < n; i += kTopThreads) s[i] = 0;
  __syncthreads();
  for (int k = 2; k <= n; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = t; i < (n >> 1); i += kTopThreads) {
        const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
        const uint64_t x = s[a], y = s[b];
        const bool down = (a & k) == 0;
        if ((x < y) == down) {
          s[a] = y;
          s[b] = x;
        }
      }
      __syncthreads();
    }
  }
}

__device__ __forceinline__ int pow2_at_least(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

template <typename T, int U, int MINB>
__global__ void __launch_bounds__(kTopThreads, MINB) logits_topk_kernel(const T* __restrict__ logits, int64_t ld,
                                                                        int V, int K, float c, float inv_t,
                                                                        float* __restrict__ logp,
                                                                        int64_t* __restrict__ ids) {
  constexpr int kRound = U * kTopThreads;
  static_assert(kTopList >= 2 * kRound, "the list holds a round behind its limit");
  __shared__ uint64_t s_buf[kTopBuf];
  __shared__ int s_list[kTopList];
  __shared__ float s_red[64], s_part[2][8];
  __shared__ int s_cnt, s_noted;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t r = blockIdx.x / C;
  const int tid = (int)threadIdx.x;
  const RowPart<T> p(logits, ld, r, V, rank, C);

  float m = -INFINITY, s = 0.f;
  float mine = -INFINITY;  // the largest value of this thread, NaN aside
  bool any = false;        // this thread had a column
  uint64_t bar = 0;        // keys at or below it are out
  float bar_value = -INFINITY;

  // Columns of the noted groups above the bar into the buffer.
  auto work_off = [&]() {
    __syncthreads();
    const int n = s_noted;
    for (int b = 0; b < n; b += kTopThreads) {
      Group8<T> g;
      int v0 = 0;
      uint32_t pend = 0;
      auto key_of = [&](int k) {
        return ((uint64_t)value_key(g.get(k)) << 32) | (0xffffffffu - (uint32_t)(v0 + k));
      };
      if (b + tid < n) {
        const int j = s_list[b + tid];
        load_group(g, p.rv, j);
        v0 = p.rv.first(j);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (v0 + k >= 0 && v0 + k < V && key_of(k) > bar) pend |= 1u << k;
      }
      while (true) {
        if (pend) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (!((pend >> k) & 1u)) continue;
            const int at = atomicAdd(&s_cnt, 1);
            if (at < kTopBuf) {
              s_buf[at] = key_of(k);
              pend &= ~(1u << k);
            }
          }
        }
        if (!__syncthreads_or(pend != 0)) break;
        // The buffer is full: keep its K largest, raise the bar, and try again with what is left.
        sort_keys(s_buf, kTopBuf, kTopBuf);
        bar = s_buf[K - 1];
        bar_value = key_value((uint32_t)(bar >> 32));
        if (tid == 0) s_cnt = K;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (((pend >> k) & 1u) && key_of(k) <= bar) pend &= ~(1u << k);
        __syncthreads();
      }
    }
    __syncthreads();
    if (tid == 0) s_noted = 0;
    __syncthreads();
  };
  // Raise the bar to the largest value (16 bits of its key) that at least K threads' maxima reach.
  auto raise_bar = [&]() {
    const uint32_t key = any ? value_key(mine) : 0u;
    uint32_t t = 0;
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t cand = t | (1u << bit);
      if (__syncthreads_count(key >= cand) >= K) t = cand;
    }
    const uint64_t found = t > 0 ? ((uint64_t)t << 32) - 1 : 0;  // values equal to it stay in
    if (found > bar) {
      bar = found;
      bar_value = key_value(t);
    }
  };
  // Note a group that reaches the bar; any group once a NaN or +inf came by (s is NaN then).  Returns
  // whether the list is near its end.
  auto below = [&](float top) { return top < bar_value && s == s; };
  auto note = [&](float top, int j) {
    if (below(top)) return false;
    const int at = atomicAdd(&s_noted, 1);
    if (at < kTopList) s_list[at] = j;
    return at >= kTopList - kRound - 1;
  };

  // The first sweep assumes that the list holds every noted group, and has no barrier but those of the
  // bar (after rounds 1, 3, 7, 15, ...).  Where it did not (rising rows, many equal values), a second
  // sweep looks after every round and works the list off in between.
  for (bool careful = false;; careful = true) {
    if (tid == 0) s_cnt = s_noted = 0;
    m = -INFINITY;
    s = 0.f;
    __syncthreads();
    bool full = false;
    int round = 0, next_bar = 0;
    int jb = p.a;
    for (; jb + kRound <= p.b; jb += kRound, ++round) {
      Group8<T> g[U];
#pragma unroll
      for (int u = 0; u < U; ++u) g[u].load(p.at(jb + u * kTopThreads + tid));
      float top[U];
      online_groups<T, U>(g, c, m, s, top);
      any = true;
      float mx = top[0];
#pragma unroll
      for (int u = 1; u < U; ++u) mx = fmaxf(mx, top[u]);
      mine = fmaxf(mine, mx);
      if (round == next_bar) {
        raise_bar();
        next_bar = 2 * next_bar + 2;
      }
      if (!below(mx)) {
#pragma unroll
        for (int u = 0; u < U; ++u) full |= note(top[u], jb + u * kTopThreads + tid);
      }
      if (careful && __syncthreads_or(full)) {
        work_off();
        full = false;
      }
    }
    // what is left, a group a thread at a time: whole groups, then those that reach past the row
    auto single = [&](int j) {
      Group8<T> h[1];
      float top[1] = {-INFINITY};
      if (j >= 0) {
        load_group(h[0], p.rv, j);
        online_groups<T, 1>(h, c, m, s, top);
        any = true;
        mine = fmaxf(mine, top[0]);
      }
      if (round++ == 0) raise_bar();
      if (j >= 0) full |= note(top[0], j);
      if (careful && __syncthreads_or(full)) {
        work_off();
        full = false;
      }
    };
    for (; jb < p.b; jb += kTopThreads) single(jb + tid < p.b ? jb + tid : -1);
    if (p.a > p.j0 || p.b < p.j1) single(p.edge(kTopThreads - 1 - tid));
    __syncthreads();
    if (careful || s_noted <= kTopList) break;
    __syncthreads();  // s_noted is read before it is cleared
  }
  work_off();
  block_online_merge(c, m, s, s_red);
  const int have = min(s_cnt, kTopBuf);
  sort_keys(s_buf, have, pow2_at_least(max(have, K)));
  if (C > 1) {
    // Every block's K largest go to the first one, behind its own, and are sorted there.
    cluster.sync();
    uint64_t* dst = cluster.map_shared_rank(s_buf, 0);
    if (rank > 0)
      for (int i = threadIdx.x; i < K; i += kTopThreads) dst[rank * K + i] = s_buf[i];
    if (threadIdx.x == 0) {
      float* part = cluster.map_shared_rank(&s_part[0][0], 0);
      part[rank] = m;
      part[8 + rank] = s;
    }
    cluster.sync();
    if (rank != 0) return;
    sort_keys(s_buf, C * K, pow2_at_least(C * K));
    m = -INFINITY;
    s = 0.f;
    for (int q = 0; q < C; ++q) online_merge(c, m, s, s_part[0][q], s_part[1][q]);
  }
  const float ls = log2f(s) * kLn2;
  for (int i = threadIdx.x; i < K; i += kTopThreads) {
    const uint64_t key = s_buf[i];
    const float x = key_value((uint32_t)(key >> 32));
    logp[r * K + i] = (x - m) * inv_t - ls;
    ids[r * K + i] = (int64_t)(0xffffffffu - (uint32_t)key);
  }
}

template <typename T>
int launch_topk(const void* logits, int64_t ld, int64_t N, int V, int K, float c, float inv_t, float* logp,
                int64_t* ids, cudaStream_t s) {
  const int C = row_cluster(N, V, kTopThreads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(N * C), 1, 1);
  cfg.blockDim = dim3(kTopThreads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kern = logits_topk_kernel<T, sizeof(T) == 2 ? 4 : 2, sizeof(T) == 2 ? 3 : 2>;
  IKRL_CUDA(cudaLaunchKernelEx(&cfg, kern, reinterpret_cast<const T*>(logits), ld, V, K, c, inv_t,
                               logp, ids));
  return check_launch("logits_topk_kernel");
}

}  // namespace
}  // namespace ikrl

using namespace ikrl;

extern "C" int ikrl_logits_topk(const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V, int32_t K,
                                float temperature, float* logp, int64_t* ids, void* stream) {
  clear_error();
  const char* what = "ikrl_logits_topk";
  int rc = check_logits_arg(what, logits, dtype, ld, N, V);
  if (rc) return rc;
  IKRL_REQUIRE(K >= 1 && K <= kMaxEntries, IKRL_ERR_UNSUPPORTED, "%s: K=%d outside 1..%d", what, K, kMaxEntries);
  IKRL_REQUIRE(K <= V, IKRL_ERR_INVALID_ARGUMENT, "%s: K=%d of V=%d columns", what, K, V);
  const float c = (float)(1.4426950408889634 / (double)temperature);
  const float inv_t = (float)(1.0 / (double)temperature);
  IKRL_REQUIRE(temperature > 0.f && c > 0.f && isfinite(c), IKRL_ERR_INVALID_ARGUMENT,
               "%s: temperature %g must be positive and finite", what, (double)temperature);
  if (N == 0) return IKRL_OK;
  IKRL_REQUIRE(logits && logp && ids, IKRL_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  return dtype == IKRL_DTYPE_BF16 ? launch_topk<uint16_t>(logits, ld, N, V, K, c, inv_t, logp, ids, as_stream(stream))
                                  : launch_topk<float>(logits, ld, N, V, K, c, inv_t, logp, ids, as_stream(stream));
}
