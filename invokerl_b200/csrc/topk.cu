// The k likeliest tokens of each row of logits and their log-probs over the whole vocabulary: what
// a teacher gives a distillation.
//
// One pass over the row, bound by HBM.  Beside the running logsumexp, a block notes the groups of
// eight columns whose maximum reaches a bar, a lower bound of the k-th largest value: the k-th largest
// of the threads' own maxima so far, found bit by bit with block-wide counts and raised after 1, 3,
// 7, 15, ... rounds of 16384 columns.  With 512 threads that bound is nearly the k-th largest itself,
// so of V columns in no particular order about k (1 + log2(V / 16384)) groups are noted.  They are read
// again (from L2), their columns above the last bar go to a buffer of keys, and the buffer is sorted.
// Where a list does not hold the noted groups (rising rows, many equal values) the row is swept again,
// working the list off on the way and cutting the keys to the k largest, which raises the bar to the
// k-th key itself.
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

// The lower bound that decides which groups are noted.
struct Bar {
  uint64_t key = 0;  // keys at or below it are out
  float value = -INFINITY;
  // To the largest value (16 bits of its key) that at least K threads' maxima reach.
  __device__ __forceinline__ void raise(bool any, float mine, int K) {
    const uint32_t key_mine = any ? value_key(mine) : 0u;
    uint32_t t = 0;
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t cand = t | (1u << bit);
      if (__syncthreads_count(key_mine >= cand) >= K) t = cand;
    }
    const uint64_t found = t > 0 ? ((uint64_t)t << 32) - 1 : 0;  // values equal to it stay in
    if (found > key) {
      key = found;
      value = key_value(t);
    }
  }
};

// One sweep of a block over its part: the running sums, the bar, and note(j, top) for each group whose
// maximum `top` reaches it (NaN: the group may hold a NaN), then end_round() by all threads.  The bar is
// raised once more at the end: what it then leaves of the noted groups is little more than K columns.
template <typename T, int U, typename Note, typename End>
__device__ __forceinline__ void sweep_part(const RowPart<T>& p, int K, float c, float& m, float& s, Bar& bar,
                                           Note note, End end_round) {
  constexpr int kRound = U * kTopThreads;
  const int tid = (int)threadIdx.x;
  float mine = -INFINITY;  // the largest value of this thread, NaN aside
  bool any = false;        // this thread had a column
  m = -INFINITY;
  s = 0.f;
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
      bar.raise(any, mine, K);
      next_bar = 2 * next_bar + 2;
    }
    // any group counts once a NaN or +inf came by (s is NaN then)
    if (!(mx < bar.value && s == s)) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (!(top[u] < bar.value && s == s)) note(jb + u * kTopThreads + tid, s == s ? top[u] : nan_f32());
    }
    end_round();
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
    if (round++ == 0) bar.raise(any, mine, K);
    if (j >= 0 && !(top[0] < bar.value && s == s)) note(j, s == s ? top[0] : nan_f32());
    end_round();
  };
  for (; jb < p.b; jb += kTopThreads) single(jb + tid < p.b ? jb + tid : -1);
  if (p.a > p.j0 || p.b < p.j1) single(p.edge(kTopThreads - 1 - tid));
  if (round > 2) bar.raise(any, mine, K);
}

// Columns of the groups list[0, n) above the bar into the buffer of keys (s_cnt of them).
template <typename T>
__device__ __forceinline__ void absorb(const RowView<T>& rv, const int* list, int n, int K, Bar& bar, uint64_t* s_buf,
                                       int* s_cnt) {
  const int tid = (int)threadIdx.x;
  for (int b = 0; b < n; b += kTopThreads) {
    Group8<T> g;
    int v0 = 0;
    uint32_t pend = 0;
    auto key_of = [&](int k) {
      return ((uint64_t)value_key(g.get(k)) << 32) | (0xffffffffu - (uint32_t)(v0 + k));
    };
    if (b + tid < n) {
      const int j = list[b + tid];
      load_group(g, rv, j);
      v0 = rv.first(j);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (v0 + k >= 0 && v0 + k < rv.V && key_of(k) > bar.key) pend |= 1u << k;
    }
    while (true) {
      if (pend) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (!((pend >> k) & 1u)) continue;
          const int at = atomicAdd(s_cnt, 1);
          if (at < kTopBuf) {
            s_buf[at] = key_of(k);
            pend &= ~(1u << k);
          }
        }
      }
      if (!__syncthreads_or(pend != 0)) break;
      // The buffer is full: keep its K largest, raise the bar, and try again with what is left.
      sort_keys(s_buf, kTopBuf, kTopBuf);
      bar.key = s_buf[K - 1];
      bar.value = key_value((uint32_t)(bar.key >> 32));
      if (tid == 0) *s_cnt = K;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (((pend >> k) & 1u) && key_of(k) <= bar.key) pend &= ~(1u << k);
      __syncthreads();
    }
  }
}

struct TopShared {
  uint64_t buf[kTopBuf];
  int list[kTopList];
  float red[64];
  float m, s;
  int cnt, noted;
};

// A block's part of a row: its sums and, in sh.buf, keys (their number is returned, at most `limit`) that
// hold its K largest, in no order.  The first sweep assumes that the list holds every noted group and has no barrier but those of the bar;
// where it did not, a second one looks after every round and works the list off in between.
template <typename T, int U>
__device__ __forceinline__ int part_topk(const RowPart<T>& p, int K, float c, int limit, float& m, float& s,
                                         TopShared& sh) {
  constexpr int kRound = U * kTopThreads;
  static_assert(kTopList >= 2 * kRound, "the list holds a round behind its limit");
  const int tid = (int)threadIdx.x;
  Bar bar;
  auto work_off = [&]() {
    __syncthreads();
    absorb(p.rv, sh.list, sh.noted, K, bar, sh.buf, &sh.cnt);
    __syncthreads();
    if (tid == 0) sh.noted = 0;
    __syncthreads();
  };
  for (bool careful = false;; careful = true) {
    if (tid == 0) sh.cnt = sh.noted = 0;
    __syncthreads();
    bool full = false;
    sweep_part<T, U>(
        p, K, c, m, s, bar,
        [&](int j, float) {
          const int at = atomicAdd(&sh.noted, 1);
          if (at < kTopList) sh.list[at] = j;
          full |= at >= kTopList - kRound - 1;
        },
        [&]() {
          if (careful && __syncthreads_or(full)) {
            work_off();
            full = false;
          }
        });
    __syncthreads();
    if (careful || sh.noted <= kTopList) break;
    __syncthreads();  // noted is read before it is cleared
  }
  work_off();
  block_online_merge(c, m, s, sh.red);
  if (tid == 0) {  // one thread's rounding for all: which thread writes an output depends on timing
    sh.m = m;
    sh.s = s;
  }
  __syncthreads();
  m = sh.m;
  s = sh.s;
  const int have = min(sh.cnt, kTopBuf);
  if (have <= limit) return have;
  sort_keys(sh.buf, have, pow2_at_least(have));
  return K;
}

// The K largest of n keys (n >= K) as a row's output: a key's place is the number of keys above it.
template <int THREADS>
__device__ __forceinline__ void write_topk(const uint64_t* keys, int n, int K, float m, float s, float inv_t,
                                           float* __restrict__ logp, int64_t* __restrict__ ids) {
  const float ls = log2f(s) * kLn2;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const uint64_t key = keys[i];
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) place += keys[j] > key;
    if (place >= K) continue;
    const float x = key_value((uint32_t)(key >> 32));
    logp[place] = (x - m) * inv_t - ls;
    ids[place] = (int64_t)(0xffffffffu - (uint32_t)key);
  }
}

// Few rows: one launch, a cluster of blocks a row (one block when it is short).
template <typename T, int U>
__global__ void __launch_bounds__(kTopThreads, 2) logits_topk_kernel(const T* __restrict__ logits, int64_t ld, int V,
                                                                     int K, float c, float inv_t,
                                                                     float* __restrict__ logp,
                                                                     int64_t* __restrict__ ids) {
  __shared__ TopShared sh;
  __shared__ float s_part[2][8];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t r = blockIdx.x / C;
  const RowPart<T> p(logits, ld, r, V, rank, C);
  __shared__ int s_have[8];
  float m, s;
  int have = part_topk<T, U>(p, K, c, kTopBuf / C, m, s, sh);
  if (C > 1) {
    // Every block's keys go to the first one, behind those of the blocks before it.
    cluster.sync();
    if (threadIdx.x < C) cluster.map_shared_rank(s_have, threadIdx.x)[rank] = have;
    if (threadIdx.x == 0) {
      float* part = cluster.map_shared_rank(&s_part[0][0], 0);
      part[rank] = m;
      part[8 + rank] = s;
    }
    cluster.sync();
    int before = 0, total = 0;
    for (int q = 0; q < C; ++q) {
      before += q < rank ? s_have[q] : 0;
      total += s_have[q];
    }
    if (rank > 0) {
      uint64_t* dst = cluster.map_shared_rank(sh.buf, 0);
      for (int i = threadIdx.x; i < have; i += kTopThreads) dst[before + i] = sh.buf[i];
    }
    cluster.sync();
    if (rank != 0) return;
    have = total;
    m = -INFINITY;
    s = 0.f;
    for (int q = 0; q < C; ++q) online_merge(c, m, s, s_part[0][q], s_part[1][q]);
  }
  write_topk<kTopThreads>(sh.buf, have, K, m, s, inv_t, logp + r * K, ids + r * K);
}

// Many rows.  One launch sweeps parts of rows and leaves, per part, its sums, its bar and the groups it
// noted; blocks end with the sweep, so the memory never waits for a choice.  The next picks each row's K
// largest out of the noted groups, all rows at once, and a last one takes the rows (hardly any) whose
// lists did not hold them.
struct TopNotes {
  int2* list;     // [N parts][kNoteCap] group and its maximum
  int* count;     // [N parts] noted groups; above kNoteCap: some are missing, the row is swept again
  uint64_t* bar;  // [N parts]
  float* part;    // [2][N parts] maxima and sums
};
constexpr int kNoteCap = 2048;

inline size_t top_notes_bytes(int64_t parts) {
  auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
  return al((size_t)parts * kNoteCap * 8) + al((size_t)parts * 4) + 2 * al((size_t)parts * 8);
}
inline TopNotes top_notes(void* ws, int64_t parts) {
  auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
  char* p = reinterpret_cast<char*>(ws);
  TopNotes t;
  t.list = reinterpret_cast<int2*>(p); p += al((size_t)parts * kNoteCap * 8);
  t.count = reinterpret_cast<int*>(p); p += al((size_t)parts * 4);
  t.bar = reinterpret_cast<uint64_t*>(p); p += al((size_t)parts * 8);
  t.part = reinterpret_cast<float*>(p);
  return t;
}

template <typename T, int U, int MINB>
__global__ void __launch_bounds__(kTopThreads, MINB) topk_note_kernel(const T* __restrict__ logits, int64_t ld, int V,
                                                                      int K, int segs, float c, int64_t parts,
                                                                      TopNotes notes) {
  __shared__ float s_red[64];
  __shared__ int s_noted;
  const int64_t q = blockIdx.x, r = q / segs;
  const RowPart<T> p(logits, ld, r, V, (int)(q - r * segs), segs);
  if (threadIdx.x == 0) s_noted = 0;
  __syncthreads();
  Bar bar;
  float m, s;
  int2* list = notes.list + q * kNoteCap;
  sweep_part<T, U>(
      p, K, c, m, s, bar,
      [&](int j, float top) {
        const int at = atomicAdd(&s_noted, 1);
        if (at < kNoteCap) list[at] = make_int2(j, __float_as_int(top));
      },
      []() {});
  block_online_merge(c, m, s, s_red);  // its barrier also closes s_noted
  if (threadIdx.x == 0) {
    notes.count[q] = s_noted;
    notes.bar[q] = bar.key;
    notes.part[q] = m;
    notes.part[parts + q] = s;
  }
}

// A row's K largest out of its noted groups.  Rows with missing groups, or with more columns above the bar
// than the buffer holds, are left to topk_again_kernel: their first part's count says so.
constexpr int kSelectThreads = 256;
constexpr int kSelectBuf = 2048;
template <typename T>
__global__ void __launch_bounds__(kSelectThreads) topk_select_kernel(const T* __restrict__ logits, int64_t ld, int V,
                                                                     int K, int segs, float c, float inv_t,
                                                                     int64_t parts, TopNotes notes,
                                                                     float* __restrict__ logp,
                                                                     int64_t* __restrict__ ids) {
  __shared__ uint64_t s_buf[kSelectBuf];
  __shared__ int s_cnt;
  const int64_t r = blockIdx.x, q0 = r * segs;
  if (threadIdx.x == 0) s_cnt = 0;
  float m = -INFINITY, s = 0.f;
  uint64_t bar = 0;
  bool missing = false;
  for (int q = 0; q < segs; ++q) {
    online_merge(c, m, s, notes.part[q0 + q], notes.part[parts + q0 + q]);
    bar = max(bar, notes.bar[q0 + q]);  // each is below the K-th largest of its part
    missing |= notes.count[q0 + q] > kNoteCap;
  }
  if (missing) {
    if (threadIdx.x == 0) notes.count[q0] = kNoteCap + 1;
    return;
  }
  __syncthreads();
  const RowView<T> rv(logits, ld, r, V);
  for (int q = 0; q < segs; ++q) {
    const int n = notes.count[q0 + q];
    for (int i = threadIdx.x; i < n; i += kSelectThreads) {
      const int2 note = notes.list[(q0 + q) * kNoteCap + i];
      const float top = __int_as_float(note.y);
      if (top == top && value_key(top) < (uint32_t)(bar >> 32)) continue;  // nothing in it above the bar
      Group8<T> g;
      load_group(g, rv, note.x);
      const int v0 = rv.first(note.x);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint64_t key = ((uint64_t)value_key(g.get(k)) << 32) | (0xffffffffu - (uint32_t)(v0 + k));
        if (v0 + k < 0 || v0 + k >= V || key <= bar) continue;
        const int at = atomicAdd(&s_cnt, 1);
        if (at < kSelectBuf) s_buf[at] = key;
      }
    }
  }
  __syncthreads();
  const int have = s_cnt;
  if (have > kSelectBuf) {
    if (threadIdx.x == 0) notes.count[q0] = kNoteCap + 1;
    return;
  }
  write_topk<kSelectThreads>(s_buf, have, K, m, s, inv_t, logp + r * K, ids + r * K);
}

template <typename T, int U>
__global__ void __launch_bounds__(kTopThreads, 2) topk_again_kernel(const T* __restrict__ logits, int64_t ld, int64_t N,
                                                                    int V, int K, int segs, float c, float inv_t,
                                                                    TopNotes notes, float* __restrict__ logp,
                                                                    int64_t* __restrict__ ids) {
  __shared__ TopShared sh;
  bool any = false;
  for (int64_t r = blockIdx.x + (int64_t)threadIdx.x * gridDim.x; r < N; r += (int64_t)gridDim.x * kTopThreads)
    any |= notes.count[r * segs] > kNoteCap;
  if (!__syncthreads_or(any)) return;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    if (notes.count[r * segs] <= kNoteCap) continue;
    float m, s;
    const RowPart<T> p(logits, ld, r, V, 0, 1);
    const int have = part_topk<T, U>(p, K, c, kTopBuf, m, s, sh);
    write_topk<kTopThreads>(sh.buf, have, K, m, s, inv_t, logp + r * K, ids + r * K);
    __syncthreads();
  }
}

template <typename T> constexpr int top_unroll() { return sizeof(T) == 2 ? 4 : 2; }
constexpr int64_t kTopFew = 2 * kNumSMs;  // rows up to which one launch with clusters takes them

int top_parts(int64_t N, int V, int dtype) {
  return dtype == IKRL_DTYPE_BF16 ? row_parts(N, V, 2, kTopThreads * top_unroll<uint16_t>())
                                  : row_parts(N, V, 4, kTopThreads * top_unroll<float>());
}

template <typename T>
int launch_topk(const void* logits, int64_t ld, int64_t N, int V, int K, float c, float inv_t, float* logp,
                int64_t* ids, void* ws, int segs, cudaStream_t s) {
  constexpr int U = top_unroll<T>();
  const T* x = reinterpret_cast<const T*>(logits);
  if (N > kTopFew) {
    const int64_t parts = N * segs;
    const TopNotes notes = top_notes(ws, parts);
    topk_note_kernel<T, U, 3><<<(unsigned)parts, kTopThreads, 0, s>>>(x, ld, V, K, segs, c, parts, notes);
    int rc = check_launch("topk_note_kernel");
    if (rc) return rc;
    topk_select_kernel<T><<<(unsigned)N, kSelectThreads, 0, s>>>(x, ld, V, K, segs, c, inv_t, parts, notes, logp, ids);
    if ((rc = check_launch("topk_select_kernel"))) return rc;
    topk_again_kernel<T, U><<<2 * kNumSMs, kTopThreads, 0, s>>>(x, ld, N, V, K, segs, c, inv_t, notes, logp, ids);
    return check_launch("topk_again_kernel");
  }
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
  auto kern = logits_topk_kernel<T, U>;
  IKRL_CUDA(cudaLaunchKernelEx(&cfg, kern, x, ld, V, K, c, inv_t, logp, ids));
  return check_launch("logits_topk_kernel");
}

}  // namespace
}  // namespace ikrl

using namespace ikrl;

extern "C" {

size_t ikrl_logits_topk_workspace_bytes(int32_t dtype, int64_t N, int32_t V) {
  if (N <= kTopFew || V <= 0) return 0;
  return top_notes_bytes(N * top_parts(N, V, dtype));
}

int ikrl_logits_topk(const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V, int32_t K,
                     float temperature, float* logp, int64_t* ids, void* ws, size_t ws_bytes, void* stream) {
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
  int segs = 1;
  if (N > kTopFew) {
    segs = top_parts(N, V, dtype);
    while (segs * K > kSelectBuf / 2) segs /= 2;  // each part may leave a little more than K keys
    IKRL_REQUIRE(N * segs <= 0x7fffffffLL, IKRL_ERR_UNSUPPORTED, "%s: N=%lld rows of V=%d need too many blocks", what,
                 (long long)N, V);
    const size_t need = top_notes_bytes(N * segs);
    IKRL_REQUIRE(ws != nullptr && ws_bytes >= need, IKRL_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", what, ws_bytes,
                 need);
    IKRL_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 255) == 0, IKRL_ERR_ALIGNMENT,
                 "%s: workspace must be 256-byte aligned", what);
  }
  return dtype == IKRL_DTYPE_BF16
             ? launch_topk<uint16_t>(logits, ld, N, V, K, c, inv_t, logp, ids, ws, segs, as_stream(stream))
             : launch_topk<float>(logits, ld, N, V, K, c, inv_t, logp, ids, ws, segs, as_stream(stream));
}

}  // extern "C"
