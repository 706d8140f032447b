// The k likeliest tokens of each row of logits and their log-probs over the whole vocabulary: what
// a teacher gives a distillation.
//
// One pass over the row, bound by HBM.  Beside the running logsumexp a thread keeps the largest value of
// each of its rounds (U groups of eight columns) in shared memory.  Behind up to kTopRounds rounds a bar is
// set, a lower bound of the K-th largest value: the K-th largest of the threads' own maxima (of 512, so it
// is nearly the K-th largest itself: in a random order 512 ln(512 / (512 - K)) columns reach it).  The rounds
// whose maximum reaches the bar are read again, from L2, and their columns above it go to a buffer of keys.
// Where the buffer fills (many equal values) it is sorted and cut to its K largest, which raises the bar
// to the K-th key itself.
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

constexpr int kTopThreads = 512;  // threads that sweep
constexpr int kTopBuf = 2048;     // keys of the buffer
constexpr int kTopRounds = 12;    // rounds between two bars
constexpr int kTopList = 1024;    // rounds to be read again at a time
static_assert(kTopBuf >= 8 * kMaxEntries, "the buffer holds K keys of each block of a cluster");
static_assert(kTopRounds * kTopThreads < 0xfffe, "list entries are 16 bits");

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
__device__ __forceinline__ uint16_t key16(float x) { return (uint16_t)(value_key(x) >> 16); }

__device__ __forceinline__ int pow2_at_least(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
  asm volatile("barrier.cta.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// N threads from thread FROM of the block on that choose keys together, with barrier ID.
template <int FROM, int N_, int ID>
struct Team {
  static constexpr int N = N_;
  static __device__ __forceinline__ int tid() { return (int)threadIdx.x - FROM; }
  static __device__ __forceinline__ void sync() {
    asm volatile("barrier.cta.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
  }
  static __device__ __forceinline__ bool any(bool x) {
    int r;
    asm volatile(
        "{\n.reg .pred a, b;\nsetp.ne.s32 a, %1, 0;\nbarrier.cta.red.or.pred b, %2, %3, a;\n"
        "selp.s32 %0, 1, 0, b;\n}"
        : "=r"(r)
        : "r"((int)x), "n"(ID), "n"(N)
        : "memory");
    return r != 0;
  }
};

// Sort s[0, n) descending (bitonic), n a power of two; the keys behind `have` count as 0.
template <typename Tm>
__device__ __forceinline__ void sort_keys(uint64_t* s, int have, int n) {
  for (int i = have + Tm::tid(); i < n; i += Tm::N) s[i] = 0;
  Tm::sync();
  for (int k = 2; k <= n; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = Tm::tid(); i < (n >> 1); i += Tm::N) {
        const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
        const uint64_t x = s[a], y = s[b];
        if ((x < y) == ((a & k) == 0)) {
          s[a] = y;
          s[b] = x;
        }
      }
      // pairs up to 32 apart lie in the 64 keys that a warp exchanges
      if (j > 32 || (j == 1 && (k >= 64 || k == n))) Tm::sync();
      else __syncwarp();
    }
  }
}

// The largest t that at least K of a warp's 16-bit values v[N] of each lane reach: bit by bit behind the
// bits that all of them share.  At least K values.
template <int N>
__device__ __forceinline__ uint32_t kth_of_warp(const uint32_t (&v)[N], int K) {
  uint32_t any = 0, all = 0xffffu;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    any |= v[i];
    all &= v[i];
  }
  any = __reduce_or_sync(0xffffffffu, any);
  all = __reduce_and_sync(0xffffffffu, all);
  uint32_t bit = any ^ all;  // of these the highest
  bit = bit ? 1u << (31 - __clz(bit)) : 0u;
  uint32_t t = bit ? all & ~(2 * bit - 1) : all;
  for (; bit; bit >>= 1) {
    const uint32_t cand = t | bit;
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) cnt += v[i] >= cand;
    if (__reduce_add_sync(0xffffffffu, cnt) >= K) t = cand;
  }
  return t;
}

// What a sweep leaves of up to kTopRounds rounds.
struct TopSweep {
  uint16_t top[kTopRounds * kTopThreads];  // key16 of each round's maximum; NaN once one (or +inf) came by
  uint16_t mine[kTopThreads];              // key16 of the threads' maxima so far in this row
  float m[kTopThreads / 32], s[kTopThreads / 32];
};

template <typename Tm>
struct TopKeys {
  uint64_t key[kTopBuf];
  uint16_t list[kTopList + 8 * Tm::N];  // round * kTopThreads + thread, or 0xfffe + t for edge t
  int cnt, listed;
  uint32_t kth;
};

// The lower bound that decides which columns come into question.
struct Bar {
  uint64_t key = 0;  // keys at or below it are out
  float value = -INFINITY;
  __device__ __forceinline__ void raise(uint64_t to, float v) {
    if (to > key) {
      key = to;
      value = v;
    }
  }
};

// One round: the running sums, and its largest value.  done(u): see online_groups.
template <typename T, int U, typename Done>
__device__ __forceinline__ uint16_t sweep_round(Group8<T> (&g)[U], float c, float& m, float& s, float& mine,
                                                Done done) {
  float top[U];
  online_groups<T, U>(g, c, m, s, top, done);
  float mx = top[0];
#pragma unroll
  for (int u = 1; u < U; ++u) mx = fmaxf(mx, top[u]);
  mine = fmaxf(mine, mx);
  return s == s ? key16(mx) : (uint16_t)0xffff;
}

// Groups that reach past the row (p.edge), by the last two of the threads that sweep.
template <typename T>
__device__ __forceinline__ void sweep_edge(const RowPart<T>& p, float c, float& m, float& s, float& mine) {
  const int j = p.edge(kTopThreads - 1 - (int)threadIdx.x);
  if (j < 0) return;
  Group8<T> g[1];
  load_group(g[0], p.rv, j);
  float top[1];
  online_groups<T, 1>(g, c, m, s, top, [](int) {});
  mine = fmaxf(mine, top[0]);
}

template <int N>
__device__ __forceinline__ void warp_online_merge(float c, float& m, float& s) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1)
    online_merge(c, m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
}

// Word i of w, without memory.
template <int N>
__device__ __forceinline__ uint32_t pick(const uint32_t (&w)[N], int i) {
  uint32_t x = w[0];
#pragma unroll
  for (int k = 1; k < N; ++k) x = i == k ? w[k] : x;
  return x;
}

// Columns above the bar of the n listed rounds into the buffer of keys, a round a thread.  start: first group
// of round 0.
template <typename Tm, typename T, int U>
__device__ __forceinline__ void absorb(const RowPart<T>& p, int start, int n, int K, Bar& bar, TopKeys<Tm>& keys) {
  constexpr int W = sizeof(T) == 2 ? 4 : 8;  // words of a group
  const int tid = Tm::tid();
  for (int b = 0; b < n; b += Tm::N) {
    uint32_t w[U * W];
    uint32_t pend = 0;
    const bool on = b + tid < n;
    const int e = on ? keys.list[b + tid] : 0;
    int j0 = start + e / kTopThreads * (U * kTopThreads) + e % kTopThreads, j1 = on ? p.b : 0;
    Group8<T> g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j0 + u * kTopThreads < j1) g[u].load(p.at(j0 + u * kTopThreads));
      else g[u].fill();
    }
    if (e >= 0xfffe) {
      j0 = p.edge(e - 0xfffe);
      j1 = j0 + 1;
      load_group(g[0], p.rv, j0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < 8; ++k)  // a NaN counts
        pend |= (j0 + u * kTopThreads < j1 && !(g[u].get(k) < bar.value) ? 1u : 0u) << (8 * u + k);
#pragma unroll
      for (int i = 0; i < W; ++i) w[u * W + i] = g[u].w[i];
    }
    while (true) {
      for (; pend; pend &= pend - 1) {
        const int i = __ffs(pend) - 1;
        const int v = p.rv.first(j0 + (i >> 3) * kTopThreads) + (i & 7);
        float x;
        if constexpr (sizeof(T) == 2) {
          const uint32_t two = pick(w, i >> 1);
          x = (i & 1) ? bf16hi(two) : bf16lo(two);
        } else {
          x = __uint_as_float(pick(w, i));
        }
        const uint64_t key = ((uint64_t)value_key(x) << 32) | (0xffffffffu - (uint32_t)v);
        if (v < 0 || v >= p.rv.V || key <= bar.key) continue;
        const int at = atomicAdd(&keys.cnt, 1);
        if (at >= kTopBuf) break;
        keys.key[at] = key;
      }
      if (!Tm::any(pend != 0)) break;
      // The buffer is full: keep its K largest, raise the bar, and try again with what is left.
      sort_keys<Tm>(keys.key, kTopBuf, kTopBuf);
      const uint64_t kth = keys.key[K - 1];
      bar.raise(kth, key_value((uint32_t)(kth >> 32)));
      if (tid == 0) keys.cnt = K;
      Tm::sync();
    }
  }
}

// The columns that come into question of n swept rounds from group `start` on; `edges` with the edges of the
// part.  The caller's barrier lies before it.
template <typename Tm, typename T, int U>
__device__ __forceinline__ void choose(const RowPart<T>& p, int start, int n, bool edges, int K, Bar& bar,
                                       const TopSweep& sw, TopKeys<Tm>& keys) {
  const int tid = Tm::tid();
  if (tid < 32) {
    const uint4* mine = reinterpret_cast<const uint4*>(sw.mine) + 2 * tid;
    const uint4 a = mine[0], b = mine[1];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    static_assert(kTopThreads == 32 * 16, "a warp reads all threads' maxima");
    uint32_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = (i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
    const uint32_t t = kth_of_warp(v, K);
    if (tid == 0) keys.kth = t;
  }
  Tm::sync();
  if (const uint32_t t = keys.kth << 16; t > 0)
    bar.raise(((uint64_t)t << 32) - 1, key_value(t));  // values equal to it stay in
  if (edges && tid < 2 && p.edge(tid) >= 0) keys.list[atomicAdd(&keys.listed, 1)] = (uint16_t)(0xfffe + tid);
  // Eight rounds' maxima a thread at a time; a warp numbers those that reach the bar.
  const uint4* eight = reinterpret_cast<const uint4*>(sw.top);
  const int lane = tid & 31, steps = n * (kTopThreads / 8);
  static_assert(kTopThreads / 8 % 32 == 0, "whole warps");
  int at = tid - lane;
  bool more;
  do {
    const uint32_t least = (uint32_t)((bar.key + 1) >> 48);
    for (; at < steps; at += Tm::N) {
      const uint4 q = eight[at + lane];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
      uint32_t hit = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hit |= ((w[i] & 0xffffu) >= least ? 1u : 0u) << (2 * i);
        hit |= ((w[i] >> 16) >= least ? 2u : 0u) << (2 * i);
      }
      const int cnt = __popc(hit);
      int sum = cnt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const int total = __shfl_sync(0xffffffffu, sum, 31);
      if (total == 0) continue;
      int slot = 0;
      if (lane == 0) slot = *(volatile int*)&keys.listed >= kTopList ? -1 : atomicAdd(&keys.listed, total);
      slot = __shfl_sync(0xffffffffu, slot, 0);
      if (slot < 0) break;  // the list is full: a step a warp may come on top of it
      for (slot += sum - cnt; hit; hit &= hit - 1)
        keys.list[slot++] = (uint16_t)(8 * (at + lane) + __ffs(hit) - 1);
    }
    more = Tm::any(at < steps);
    absorb<Tm, T, U>(p, start, keys.listed, K, bar, keys);
    Tm::sync();
    if (tid == 0) keys.listed = 0;
    Tm::sync();
  } while (more);
}

// The K largest of n keys (n >= K) as a row's output.  A few keys are placed by counting the keys above each.
template <typename Tm>
__device__ __forceinline__ void write_topk(uint64_t* key, int n, int K, float m, float s, float inv_t,
                                           float* __restrict__ logp, int64_t* __restrict__ ids) {
  const float ls = log2f(s) * kLn2;
  auto put = [&](int place, uint64_t k) {
    logp[place] = (key_value((uint32_t)(k >> 32)) - m) * inv_t - ls;
    ids[place] = (int64_t)(0xffffffffu - (uint32_t)k);
  };
  if (n * ((n + Tm::N - 1) / Tm::N) <= 320) {
    for (int i = Tm::tid(); i < n; i += Tm::N) {
      const uint64_t k = key[i];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) place += key[j] > k;
      if (place < K) put(place, k);
    }
    return;
  }
  sort_keys<Tm>(key, n, pow2_at_least(n));
  for (int i = Tm::tid(); i < K; i += Tm::N) put(i, key[i]);
}

// A block a row, or a cluster of blocks where there are few rows; the block that swept chooses.
template <typename T, int U>
__global__ void __launch_bounds__(kTopThreads, 3) topk_block_kernel(const T* __restrict__ logits, int64_t ld, int V,
                                                                  int K, float c, float inv_t,
                                                                  float* __restrict__ logp,
                                                                  int64_t* __restrict__ ids) {
  using Block = Team<0, kTopThreads, 0>;
  constexpr int kRound = U * kTopThreads;
  __shared__ __align__(16) TopSweep sw;
  __shared__ TopKeys<Block> keys;
  __shared__ float s_red[64], s_part[2][8];
  __shared__ int s_have[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = (int)threadIdx.x;
  const int64_t r = blockIdx.x / C;
  const RowPart<T> p(logits, ld, r, V, rank, C);
  if (tid == 0) keys.cnt = keys.listed = 0;
  Bar bar;
  float m = -INFINITY, s = 0.f, mine = -INFINITY;
  sweep_edge(p, c, m, s, mine);
  int jb = p.a;
  do {
    const int start = jb;
    int n = 0;
    for (; n < kTopRounds && jb < p.b; ++n, jb += kRound) {
      Group8<T> g[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jb + u * kTopThreads + tid;
        if (j < p.b) g[u].load(p.at(j));
        else g[u].fill();
      }
      sw.top[n * kTopThreads + tid] = sweep_round<T, U>(g, c, m, s, mine, [](int) {});
    }
    sw.mine[tid] = key16(mine);
    Block::sync();
    choose<Block, T, U>(p, start, n, start == p.a, K, bar, sw, keys);
  } while (jb < p.b);
  block_online_merge(c, m, s, s_red);
  if (tid == 0) {  // one thread's rounding for all: which thread writes an output depends on timing
    s_part[0][0] = m;
    s_part[1][0] = s;
  }
  __syncthreads();
  int have = keys.cnt;
  if (C == 1) {
    write_topk<Block>(keys.key, have, K, s_part[0][0], s_part[1][0], inv_t, logp + r * K, ids + r * K);
    return;
  }
  if (have > kTopBuf / C) {
    sort_keys<Block>(keys.key, have, pow2_at_least(have));
    have = K;
  }
  m = s_part[0][0];
  s = s_part[1][0];
  // Every block's keys go to the first one, behind those of the blocks before it.
  cluster.sync();
  if (tid < C) cluster.map_shared_rank(s_have, tid)[rank] = have;
  if (tid == 0) {
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
    uint64_t* dst = cluster.map_shared_rank(keys.key, 0);
    for (int i = tid; i < have; i += kTopThreads) dst[before + i] = keys.key[i];
  }
  cluster.sync();
  if (rank != 0) return;
  m = -INFINITY;
  s = 0.f;
  for (int q = 0; q < C; ++q) online_merge(c, m, s, s_part[0][q], s_part[1][q]);
  if (total > kMaxEntries) {  // what lies below the K-th largest of all (16 bits of it) goes first
    uint64_t own[kTopBuf / kTopThreads];
#pragma unroll
    for (int i = 0; i < kTopBuf / kTopThreads; ++i) {
      const bool ok = i * kTopThreads + tid < total;
      own[i] = ok ? keys.key[i * kTopThreads + tid] : 0;
    }
    uint32_t t = 0;
    for (int bit = 15; bit >= 0; --bit) {
      const uint64_t cand = (uint64_t)(t | (1u << bit)) << 48;
      int reach = 0;
#pragma unroll
      for (int i = 0; i < kTopBuf / kTopThreads; ++i)
        if (i * kTopThreads < total) reach += __syncthreads_count(own[i] >= cand);
      if (reach >= K) t |= 1u << bit;
    }
    if (tid == 0) keys.cnt = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTopBuf / kTopThreads; ++i)
      if (own[i] != 0 && own[i] >= ((uint64_t)t << 48)) keys.key[atomicAdd(&keys.cnt, 1)] = own[i];
    __syncthreads();
    total = keys.cnt;
  }
  write_topk<Block>(keys.key, total, K, m, s, inv_t, logp + r * K, ids + r * K);
}

// Many rows: resident blocks take row after row.  512 threads sweep and never stop for a choice: they hand
// what they swept to 128 more, which choose and write the row's output while the next row is read.  Two
// buffers between them; barriers 2, 3 say that one is full, 4, 5 that it is free.  Top 64 of 4096 rows of
// 151936 bf16 columns: 247 us in a row of calls, 256 from a cold L2, 270 after other work (4.6 to 5.0 TB/s), nearly
// all of it the sweep, where exponentials (67% of the special function units' rate) and loads take turns; of
// 2048 fp32 rows 194 us (6.4 TB/s).
constexpr int kChoosers = 128;
constexpr int kStreamThreads = kTopThreads + kChoosers;
template <typename T, int U>
__global__ void __launch_bounds__(kStreamThreads, 2) topk_stream_kernel(const T* __restrict__ logits, int64_t ld, int64_t N,
                                                                    int V, int K, float c, float inv_t,
                                                                    float* __restrict__ logp,
                                                                    int64_t* __restrict__ ids) {
  using Choosers = Team<kTopThreads, kChoosers, 1>;
  constexpr int kRound = U * kTopThreads;
  __shared__ __align__(16) TopSweep sw[2];
  __shared__ TopKeys<Choosers> keys;
  const int tid = (int)threadIdx.x;
  if (tid < kTopThreads) {
    // g holds the next round: `left` groups from `src` (this thread's) to the end of its row
    Group8<T> g[U];
    const T* src = logits;
    int left = 0;
    auto load = [&](int u) {
      if (left >= kRound) g[u].load(src + u * kTopThreads * 8);
      else if (u * kTopThreads + tid < left) g[u].load(src + u * kTopThreads * 8);
      else g[u].fill();
    };
    auto turn_to = [&](int64_t r) {
      left = 0;
      if (r >= N) return;
      const RowPart<T> p(logits, ld, r, V, 0, 1);
      left = p.b - p.a;
      src = p.at(p.a + tid);
    };
    turn_to(blockIdx.x);
#pragma unroll
    for (int u = 0; u < U; ++u) load(u);
    int unit = 0;
    for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
      float m = -INFINITY, s = 0.f, mine = -INFINITY;
      sweep_edge(RowPart<T>(logits, ld, r, V, 0, 1), c, m, s, mine);
      bool more = left > 0;
      const bool none = !more;
      do {
        TopSweep& out = sw[unit & 1];
        if (unit > 1) bar_sync(4 + (unit & 1), kStreamThreads);
        for (int n = 0; n < kTopRounds && more; ++n) {
          src += kRound * 8;
          left -= kRound;
          more = left > 0;
          if (!more) turn_to(r + gridDim.x);
          out.top[n * kTopThreads + tid] = sweep_round<T, U>(g, c, m, s, mine, load);
        }
        out.mine[tid] = key16(mine);
        if (!more) {
          float wm = m, ws = s;
          warp_online_merge<32>(c, wm, ws);
          if ((tid & 31) == 0) {
            out.m[tid >> 5] = wm;
            out.s[tid >> 5] = ws;
          }
        }
        bar_arrive(2 + (unit & 1), kStreamThreads);
        ++unit;
      } while (more);
      if (none) {  // no round of this row carried the next one's loads
        turn_to(r + gridDim.x);
#pragma unroll
        for (int u = 0; u < U; ++u) load(u);
      }
    }
    return;
  }
  int unit = 0;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const RowPart<T> p(logits, ld, r, V, 0, 1);
    if (tid == kTopThreads) keys.cnt = keys.listed = 0;
    Choosers::sync();
    Bar bar;
    int jb = p.a;
    while (true) {
      const TopSweep& in = sw[unit & 1];
      bar_sync(2 + (unit & 1), kStreamThreads);
      const int n = min(kTopRounds, (p.b - jb + kRound - 1) / kRound);
      choose<Choosers, T, U>(p, jb, n, jb == p.a, K, bar, in, keys);
      jb += n * kRound;
      if (jb >= p.b) break;
      bar_arrive(4 + (unit & 1), kStreamThreads);
      ++unit;
    }
    float m = sw[unit & 1].m[tid & 15], s = sw[unit & 1].s[tid & 15];
    warp_online_merge<16>(c, m, s);
    m = __shfl_sync(0xffffffffu, m, 0);  // one rounding for all: which thread writes an output depends on timing
    s = __shfl_sync(0xffffffffu, s, 0);
    bar_arrive(4 + (unit & 1), kStreamThreads);
    ++unit;
    write_topk<Choosers>(keys.key, keys.cnt, K, m, s, inv_t, logp + r * K, ids + r * K);
    Choosers::sync();  // the keys are read
  }
}

template <typename T> constexpr int top_unroll() { return sizeof(T) == 2 ? 4 : 2; }

template <typename T>
int launch_topk(const void* logits, int64_t ld, int64_t N, int V, int K, float c, float inv_t, float* logp,
                int64_t* ids, cudaStream_t s) {
  constexpr int U = top_unroll<T>();
  const T* x = reinterpret_cast<const T*>(logits);
  // Rows that all have a resident block need no streaming (444 rows of 151936 bf16 columns, K = 64: 41 us
  // against 47; 600 rows: 59 against 53).  With many keys a row the choosers fall behind the sweep, and blocks
  // that choose themselves are as fast or faster (4096 rows of 50257 fp32 columns, K = 200: 242 us against 289;
  // 1776 rows of 151936 bf16 columns: K = 128 139 against 131, K = 256 174 against 176).
  if (N > 3 * kNumSMs && K <= 128) {
    topk_stream_kernel<T, U><<<2 * kNumSMs, kStreamThreads, 0, s>>>(x, ld, N, V, K, c, inv_t, logp, ids);
    return check_launch("topk_stream_kernel");
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
  auto kern = topk_block_kernel<T, U>;
  IKRL_CUDA(cudaLaunchKernelEx(&cfg, kern, x, ld, V, K, c, inv_t, logp, ids));
  return check_launch("topk_block_kernel");
}

}  // namespace
}  // namespace ikrl

using namespace ikrl;

extern "C" {

int ikrl_logits_topk(const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V, int32_t K,
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
  IKRL_REQUIRE(N <= 0x7fffffffLL, IKRL_ERR_UNSUPPORTED, "%s: N=%lld rows need too many blocks", what,
               (long long)N);
  return dtype == IKRL_DTYPE_BF16
             ? launch_topk<uint16_t>(logits, ld, N, V, K, c, inv_t, logp, ids, as_stream(stream))
             : launch_topk<float>(logits, ld, N, V, K, c, inv_t, logp, ids, as_stream(stream));
}

}  // extern "C"
