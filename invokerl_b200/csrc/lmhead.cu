// K1: fused LM-head log-prob on the 5th-generation tensor cores (tcgen05 + TMEM + TMA).
//
// Replaces invokerl/policy.py:124-191 (`_chunked_lm_head_ce` / `_chunk_ce_fn`: F.linear then
// -F.cross_entropy, chunk by chunk under torch.utils.checkpoint) and its autograd.
//
// Forward: logits tiles S = h W^T are produced in TMEM, 128 rows x 256 vocab columns at a time,
// and consumed in place by an epilogue that keeps an online (max, sum-exp) per row and picks out
// the target logit; the [N, V] logits never reach HBM.  Partial row statistics of each vocab
// split are merged by a small combine kernel: log p = S[target] - logsumexp(S).
//
// Backward: for each chunk of rows, the same GEMM recomputes S and its epilogue writes
// dS = g * (onehot - exp(S - lse)) in bf16 to a chunk workspace; two more tcgen05 GEMMs form
// dH = dS W (A K-major, B MN-major) and dW += dS^T h (both MN-major), the latter accumulated in
// fp32.  Only one chunk of dS exists at a time.
//
// Kernel shape (one CTA per SM, 192 threads):
//   warp 0      TMA producer: 4-stage ring of {A 128x64, B 256x64} bf16 tiles, 128B swizzle
//   warp 1      TMEM allocator + MMA issuer: tcgen05.mma M=128 N=256 K=16, f32 accumulators,
//               two accumulators (2 x 256 TMEM columns) so the epilogue of tile j overlaps the
//               MMAs of tile j+1
//   warps 2-5   epilogue: tcgen05.ld, one TMEM lane (= one output row) per thread
// Every mbarrier wait is bounded (sm100::kWaitTimeoutNs); on expiry the CTA records an error,
// drains its in-flight copies and MMAs, frees TMEM and exits.
#include "common.cuh"
#include "row_dist.cuh"
#include "sm100.cuh"

#include <cuda_fp16.h>

#include <atomic>
#include <mutex>
#include <vector>

namespace ikrl {
namespace {

using namespace sm100;

constexpr int BM = 128, BN = 256, BK = 64;
constexpr int kStages = 4;
constexpr int kThreads = 192;
constexpr int kEpiWarps = 4;
// The wide kernel runs four epilogue warps per TMEM lane quadrant, each on a quarter of the columns
// of each 256-column half of the 512-column tile (64 columns per half).
constexpr int kWideEpiWarps = 16;
constexpr int kWideGroups = kWideEpiWarps / 4;
constexpr int kWideThreads = 64 + 32 * kWideEpiWarps;
constexpr uint32_t kTileA = BM * BK * 2;  // 16 KB
constexpr uint32_t kTileB = BN * BK * 2;  // 32 KB
constexpr uint32_t kStageBytes = kTileA + kTileB;
constexpr uint32_t kSmemBytes = kStages * kStageBytes + 1024;  // + alignment slack
constexpr uint32_t kTmemCols = 2 * BN;
constexpr uint32_t kDsStageBytes = 32 * 32 * 2;  // a 32 x 32 bf16 block staged for a TMA store
constexpr uint32_t kMnAtomBytes = 64 * BK * 2;  // one 64-wide MN slab of an MN-major tile: 8 KB

// EPI_LSE_CACHED: the forward's epilogue that also fills the logit cache (its own instantiation,
// so the plain forward carries none of the cache's code).
// EPI_TAIL, EPI_DTAIL: forward and backward of the row losses (row_dist.cuh).  EPI_TAIL leaves each
// row's entry columns out and keeps the running sum of the others; EPI_DTAIL forms the gradient of the
// others.  EPI_TAIL_CACHED is EPI_TAIL that fills the logit cache.  EPI_STORE_TMA is EPI_STORE_BF16 whose
// blocks leave through TMA stores (the wide kernel only): for short reductions, where writing the output
// is most of the work.
enum Epi : int {
  EPI_LSE = 0,
  EPI_DLOGITS = 1,
  EPI_STORE_BF16 = 2,
  EPI_F32 = 3,
  EPI_LSE_CACHED = 4,
  EPI_TAIL = 5,
  EPI_DTAIL = 6,
  EPI_TAIL_CACHED = 7,
  EPI_STORE_TMA = 8
};
constexpr bool is_lse(int epi) { return epi == EPI_LSE || epi == EPI_LSE_CACHED; }
constexpr bool is_dlogits(int epi) { return epi == EPI_DLOGITS || epi == EPI_DTAIL; }
constexpr bool is_tail(int epi) { return epi == EPI_TAIL || epi == EPI_TAIL_CACHED; }
constexpr bool is_cached(int epi) { return epi == EPI_LSE_CACHED || epi == EPI_TAIL_CACHED; }
// Epilogues of the wide kernel that stage 32 x 32 bf16 blocks in shared memory for TMA stores.
constexpr bool is_staged(int epi) { return is_dlogits(epi) || is_cached(epi) || epi == EPI_STORE_TMA; }
// The epilogue whose launch rules (pacing, splits) an epilogue follows.
constexpr int epi_kind(int epi) {
  return (is_cached(epi) || is_tail(epi)) ? (int)EPI_LSE
         : epi == EPI_DTAIL               ? (int)EPI_DLOGITS
         : epi == EPI_STORE_TMA           ? (int)EPI_STORE_BF16
                                          : epi;
}
// Epilogues whose GEMM may have fp16 operands.
constexpr bool takes_f16(int epi) { return epi == EPI_F32 || epi == EPI_STORE_BF16 || epi == EPI_STORE_TMA; }
enum F32Mode : int { F32_STORE = 0, F32_ADD = 1, F32_ADD_TO_BF16 = 2 };

struct GemmParams {
  int M, N, K;            // C[M, N] = A[M, K] * B[N, K]^T
  int n_tiles;            // ceil(N / BN)
  int tiles_per_split;    // consecutive N tiles of one CTA
  int splits;             // number of N ranges (gridDim.x when split-major)
  int split_major;        // 1: blockIdx.x = split, blockIdx.y = row block; 0: the reverse
  const int64_t* ids;     // [M] target ids (LSE / DLOGITS)
  const float* lse;       // [M] (DLOGITS)
  const float* g;         // [M] upstream d loss / d logp (DLOGITS)
  float* part_m;          // [splits][M] running max, log2 units (LSE)
  float* part_s;          // [splits][M] sum of 2^(x - max) (LSE)
  float* part_t;          // [M] raw target logit, written by the split owning the target (LSE)
  uint16_t* out_bf16;     // DLOGITS: dS; STORE_BF16: output; F32 mode 2: bf16 output
  int64_t ld_bf16;
  float* out_f32;         // F32: accumulator
  int64_t ld_f32;
  int f32_mode;
  int* err;               // device error word
  int part_sets;          // LSE partial sets written (splits x column halves), set by the launcher
  int a_policy, b_policy; // L2 eviction priority of the A / B loads: 0 normal, 1 evict-last, 2 evict-first
  unsigned* lockstep;     // [npairs] tiles started per pair (zeroed per launch), or null: no pacing
  int64_t id_offset;      // first vocabulary id of W's rows (a vocab shard); 0 for the whole vocabulary
  int pace_kb, pace_lag;  // pacing: K blocks between checkpoints, checkpoints a pair may lead by
  int split_tail;         // wide kernel: how many of a tile's last K blocks run first-half-first
  int ksplits;            // wide kernel: K ranges per output tile (<= 1: one), each to its own
  int64_t ks_stride;      //   fp32 partial output, ks_stride elements apart (EPI_F32 only)
  int ds_tma;             // DLOGITS in the wide kernel: 1 = stage dS in shared memory, TMA-store it
  // Logit cache (LSE, optional): rows with slot[r] >= 0 store, per 32-column chunk, the bf16
  // numerators 2^(S log2e - m) relative to the chunk maximum m and m itself (log2 units), so the
  // backward can form dS without recomputing the logits.
  const int* slot;        // [M] cache slot of each row, -1 = not cached; null = no cache
  uint16_t* cache_q;      // [slots][ld_cache] bf16 numerators
  float* cache_m;         // [slots][n_mchunks] chunk maxima, log2 units
  int64_t ld_cache;
  int n_mchunks;
  // Row losses (TAIL, DTAIL)
  float c;                // log2(e) / temperature
  const int* m_dev;       // on the device, or null (TAIL): the LivePlan of the rows in use
  const int* row_idx;     // original row of each row, or null: itself (TAIL)
  const int* cols;        // [original rows][n_cols] entry columns ascending, then kNoEntry (TAIL)
  int n_cols;
  float* xk;              // [original rows][n_cols] logits at the entries, or null (TAIL)
  int64_t cache_cap;      // TAIL_CACHED: slots; a row's slot is its place in the launch
  int* part_c;            // [splits][M] columns of the maxima in part_m, or null (TAIL)
  int part_cap;           // sets that part_m, part_s and part_x hold (TAIL)
  float* part_x;          // [splits][M] sum of all logits, or null (TAIL)
  const float* level;     // [M] constant part of the gradient (DTAIL); lse: the row's ref, g: its coef
  uint16_t* out_lo;       // what rounding to out_bf16 leaves, itself rounded, or null (DTAIL)
  // Products of fp16 operands scaled by powers of two (the row losses' dW and dH; see RowRange)
  int f16;                // A and B are fp16 (F32, STORE_BF16, STORE_TMA); the output is (DTAIL)
  const float* out_scale; // what the output is multiplied by, one for all or (scale_rows) each row's, or null
  int scale_rows;
};

__device__ __forceinline__ bool mbar_wait_drain(uint32_t bar, uint32_t parity, int* err) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer() - t0 > kWaitTimeoutNs / 4) {
      atomicCAS(err, 0, kErrTimeoutDrain);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void st_global_v4(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What a row loss's forward over gathered rows runs with: the rows there are (known on the device only), the
// column ranges that suit that many, and the partial sets they leave.
enum LivePlan : int { LIVE_ROWS = 0, LIVE_TILES_PER_SPLIT = 1, LIVE_SPLITS = 2, LIVE_SETS = 3 };

// Rows of a launch: p.M, or for the row losses the count a kernel before left on the device.
template <int EPI>
__device__ __forceinline__ int live_rows(const GemmParams& p) {
  if constexpr (is_tail(EPI)) {
    if (p.m_dev != nullptr) return min(p.m_dev[LIVE_ROWS], p.M);
  }
  return p.M;
}
template <int EPI>
__device__ __forceinline__ int column_splits(const GemmParams& p) {
  if constexpr (is_tail(EPI)) {
    if (p.m_dev != nullptr) return p.m_dev[LIVE_SPLITS];
  }
  return p.splits;
}
template <int EPI>
__device__ __forceinline__ int split_tiles(const GemmParams& p) {
  if constexpr (is_tail(EPI)) {
    if (p.m_dev != nullptr) return p.m_dev[LIVE_TILES_PER_SPLIT];
  }
  return p.tiles_per_split;
}

// Epilogue role (warps 2..): drain accumulator tiles from TMEM, one row per thread, and apply the
// epilogue EPI.  acc_full[a] are this CTA's barriers; acc_empty[a] are the addresses the warps
// arrive on when a tile is consumed (this CTA's, or the pair leader's when cluster_arrive).
// tile_base: number of tiles this CTA consumed before this unit (accumulator ring position).
// Returns false when a wait gave up (abort).
// GROUPS: column groups; warp w drains TMEM lane quadrant w % 4 and column group (w - 2) / 4.
// SPLIT (wide tile, one accumulator): the halves complete separately (acc_full[0] when the first
// 256-column half of a tile is final, acc_full[1] for the second).  Every warp loads its columns
// of the first half into registers and releases that half (acc_empty[0]) at once, so the next
// tile's first-half MMAs start while it computes; then it does the same for the second half
// (acc_empty[1]).
// stage_smem (DLOGITS only, 0 = unused): this warp's 2 KB staging tile; the dS values of each
// 32 x 32 block are written there in the 64-byte swizzled layout of tm_store and sent to global
// memory with one TMA store per block, instead of 32 scattered row stores.
template <int EPI, int TILE_N = BN, int NBUF = 2, int GROUPS = 1, bool SPLIT = false>
__device__ __forceinline__ bool epilogue_role(const GemmParams& p, uint32_t tmem_base, int m0, int split, int t_begin,
                                              int t_end, int warp, int lane, const uint32_t (&acc_full)[2],
                                              const uint32_t (&acc_empty)[2], bool cluster_arrive,
                                              volatile int* abort_v, int tile_base = 0,
                                              const CUtensorMap* tm_store = nullptr, uint32_t stage_smem = 0,
                                              int64_t out_off = 0) {
  const int ntiles = t_end - t_begin;
  bool ok = true;
  const int q = warp & 3;  // TMEM lane quadrant this warp may access
  constexpr int kCols = TILE_N / GROUPS;  // columns of the tile this warp drains
  static_assert(!SPLIT || NBUF == 1, "split drain needs one accumulator");
  constexpr int kSegs = SPLIT ? 2 : 1;                      // column segments, drained in order
  constexpr int kSegCols = SPLIT ? TILE_N / (2 * GROUPS) : kCols;
  static_assert(!SPLIT || kSegCols % 32 == 0, "split segments are whole 32-column chunks");
  const int group = GROUPS == 1 ? 0 : (warp - 2) / 4;
  const int c_lo = group * kCols;
  const int r = q * 32 + lane;
  const int grow = m0 + r;
  const bool row_ok = grow < live_rows<EPI>(p);
  int64_t tgt = -1;
  float lse2 = 0.f, gval = 0.f;
  if constexpr (is_lse(EPI) || EPI == EPI_DLOGITS) {
    if (row_ok) tgt = p.ids[grow];
  }
  int cslot = -1;  // logit-cache slot of this row (LSE)
  bool cache_run = false;  // the warp's 32 rows have consecutive slots: one TMA store per block
  int cslot0 = 0;
  if constexpr (is_cached(EPI)) {
    if constexpr (EPI == EPI_TAIL_CACHED) {
      if (row_ok && grow < p.cache_cap) cslot = grow;  // slots go by place in the launch
    } else if (row_ok && p.slot != nullptr) {
      cslot = p.slot[grow];
    }
    cslot0 = __shfl_sync(0xffffffffu, cslot, 0);
    cache_run = stage_smem != 0 && __all_sync(0xffffffffu, cslot >= 0 && cslot == cslot0 + lane);
  }
  // TAIL: the row's next entry column at or after the columns read so far
  const int* next_col = nullptr;
  float* entry_x = nullptr;
  int next = kNoEntry, at = 0;
  float sum_x = 0.f;
  int run_c = 0;
  auto advance = [&]() { next = ++at < p.n_cols ? next_col[at] : kNoEntry; };
  if constexpr (is_tail(EPI)) {
    if (row_ok) {
      const int64_t row = p.row_idx != nullptr ? p.row_idx[grow] : grow;
      next_col = p.cols + row * p.n_cols;
      if (p.xk != nullptr) entry_x = p.xk + row * p.n_cols;
      int hi = p.n_cols;
      const int from = t_begin * TILE_N;
      while (at < hi) {
        const int mid = (at + hi) >> 1;
        if (next_col[mid] < from) at = mid + 1;
        else hi = mid;
      }
      if (at < p.n_cols) next = next_col[at];
    }
  }
  float level = 0.f;
  bool still = true;  // DTAIL: a row without a gradient, whose logits (padding may hold NaN) do not matter
  if constexpr (EPI == EPI_DTAIL) {
    if (row_ok) {
      lse2 = p.lse[grow] * p.c;
      gval = p.g[grow];
      level = p.level[grow];
      still = gval == 0.f && level == 0.f;
    }
  }
  if constexpr (EPI == EPI_DLOGITS) {
    if (row_ok) {
      lse2 = p.lse[grow] * kLog2e;
      gval = p.g[grow];
      if (tgt == -100) gval = 0.f;  // ignore_index rows have zero gradient
    }
  }
  // Column index of the target in this W (a vocab shard starts at id_offset); ignore_index rows
  // keep -100, which matches no column.
  if (tgt != -100) tgt -= p.id_offset;
  float out_scale = 1.f;
  if constexpr (takes_f16(EPI)) {
    if (p.out_scale != nullptr) out_scale = p.scale_rows ? (row_ok ? p.out_scale[grow] : 0.f) : p.out_scale[0];
  }
  float run_m = -INFINITY, run_s = 0.f, tval = 0.f;
  bool found = false;

  // A 32 x 32 block of 16-bit values leaves with one TMA store: row `lane` goes to the staging tile with
  // its 16-byte chunks in the 64-byte swizzled order; the tensor map clips rows and columns past its edges.
  auto store_block = [&](const uint32_t (&w)[16], int col, int row) {
    if (lane == 0) bulk_wait_read_all();  // the previous block's store has read the tile
    __syncwarp();
    const uint32_t row_addr = stage_smem + (uint32_t)lane * 64u;
    const uint32_t sw = ((uint32_t)lane >> 1) & 3u;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      st_shared_v4(row_addr + ((((uint32_t)k) ^ sw) << 4), w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    fence_async_shared();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(tm_store, stage_smem, col, row);
      bulk_commit();
    }
  };
  // The numerators v of a chunk whose maximum is cm into the logit cache.  They are at most 1: a row
  // loss keeps them in fp16, whose 11 bits its dS has as well (bf16's 8 would be most of its gradients'
  // error); what lies below 2^-14 of its chunk's maximum loses bits that the sums over the vocabulary
  // do not see.
  auto pack16 = [](float lo, float hi) -> uint32_t {
    if constexpr (EPI == EPI_TAIL_CACHED) return pack_f16x2(lo, hi);
    else return pack_bf16x2(lo, hi);
  };
  auto store_numerators = [&](const float* v, int col0, float cm) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 32; i += 2) w[i >> 1] = pack16(v[i], v[i + 1]);
    if (cache_run) {
      store_block(w, col0, cslot0);  // consecutive slots
    } else if (cslot >= 0) {
      uint16_t* dst = p.cache_q + (int64_t)cslot * p.ld_cache + col0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        st_global_v4(dst + 8 * k, w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    }
    if (cslot >= 0) p.cache_m[(int64_t)cslot * p.n_mchunks + (col0 >> 5)] = cm;
  };

  // The epilogue of one 32-column chunk of this thread's row, columns [col0, col0 + 32) of the
  // output (col0 < N; the chunk may end past N).  Warp-uniform control flow.
  auto chunk = [&](float* v, int col0) {
    if constexpr (takes_f16(EPI)) {
      if (p.out_scale != nullptr) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= out_scale;
      }
    }
    const int nvalid = min(32, p.N - col0);
    if constexpr (is_lse(EPI)) {
      float cm = -INFINITY;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < nvalid) cm = fmaxf(cm, v[i]);
      cm *= kLog2e;
      // Target gather without a dynamically indexed register array (which would go to local
      // memory): exactly one term is v[rel] * 1, every other term adds zero.
      const int64_t rel = tgt - col0;
      if (rel >= 0 && rel < nvalid) {
        const int rr = (int)rel;
        float acc_t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) acc_t += (i == rr) ? v[i] : 0.f;
        tval = acc_t;
        found = true;
      }
      // Numerators relative to the chunk maximum cm (in place of the logits), then the running
      // (max, sum) update; the numerators are what the logit cache stores.
      float cs = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        v[i] = i < nvalid ? fast_exp2(fmaf(v[i], kLog2e, -cm)) : 0.f;
        cs += v[i];
      }
      if (cm > run_m) {
        run_s = fmaf(run_s, fast_exp2(run_m - cm), cs);
        run_m = cm;
      } else {
        run_s = fmaf(cs, fast_exp2(cm - run_m), run_s);
      }
      if constexpr (EPI == EPI_LSE_CACHED) store_numerators(v, col0, cm);
    } else if constexpr (is_tail(EPI)) {
      if (p.part_x != nullptr) {
#pragma unroll
        for (int i = 0; i < 32; ++i) sum_x += i < nvalid ? v[i] : 0.f;
      }
      // Entries in this chunk leave it (their logits to xk, where it is given).
      while (next < col0) advance();  // entries of other warps' columns
      while (next < col0 + nvalid) {
        const int rel = next - col0;
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          x += i == rel ? v[i] : 0.f;
          v[i] = i == rel ? -INFINITY : v[i];
        }
        if (entry_x != nullptr) entry_x[at] = x;
        advance();
      }
      float cm = -INFINITY;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < nvalid) cm = fmaxf(cm, v[i]);
      if (p.part_c != nullptr && cm > run_m) {
        int at_max = 0;  // columns past N come last, so the lowest of equal ones is a column
#pragma unroll
        for (int i = 31; i >= 0; --i) at_max = v[i] == cm ? i : at_max;
        run_c = col0 + at_max;
      }
      const float from = cm == -INFINITY ? 0.f : cm;  // a chunk of entries only sums to 0
      float cs = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        v[i] = i < nvalid ? fast_exp2((v[i] - from) * p.c) : 0.f;
        cs += v[i];
      }
      if (cm > run_m) {
        run_s = fmaf(run_s, fast_exp2((run_m - cm) * p.c), cs);
        run_m = cm;
      } else {
        run_s = fmaf(cs, cm == -INFINITY ? 1.f : fast_exp2((cm - run_m) * p.c), run_s);
      }
      if constexpr (EPI == EPI_TAIL_CACHED) store_numerators(v, col0, cm);
    } else if constexpr (is_dlogits(EPI)) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        if constexpr (EPI == EPI_DTAIL) {
          v[i] = still ? 0.f : fmaf(gval, fast_exp2(fmaf(v[i], p.c, -lse2)), level);
          v[i + 1] = still ? 0.f : fmaf(gval, fast_exp2(fmaf(v[i + 1], p.c, -lse2)), level);
          w[i >> 1] = p.f16 ? pack_f16x2(v[i], v[i + 1]) : pack_bf16x2(v[i], v[i + 1]);
          continue;
        }
        const float p0 = fast_exp2(fmaf(v[i], kLog2e, -lse2));
        const float p1 = fast_exp2(fmaf(v[i + 1], kLog2e, -lse2));
        const float d0 = gval * (((int64_t)(col0 + i) == tgt ? 1.f : 0.f) - p0);
        const float d1 = gval * (((int64_t)(col0 + i + 1) == tgt ? 1.f : 0.f) - p1);
        w[i >> 1] = pack_bf16x2(d0, d1);
      }
      if constexpr (EPI == EPI_DTAIL) {
        if (p.out_lo != nullptr && row_ok) {
          uint16_t* lo = p.out_lo + (int64_t)grow * p.ld_bf16 + col0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (8 * k >= nvalid) break;
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = 8 * k + 2 * e;
              o[e] = pack_bf16x2(v[i] - bf16lo(w[i >> 1]), v[i + 1] - bf16hi(w[i >> 1]));
            }
            st_global_v4(lo + 8 * k, o[0], o[1], o[2], o[3]);
          }
        }
      }
      if (stage_smem != 0) {
        store_block(w, col0, m0 + q * 32);
      } else if (row_ok) {
        uint16_t* dst = p.out_bf16 + (int64_t)grow * p.ld_bf16 + col0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (8 * k < nvalid) st_global_v4(dst + 8 * k, w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
      }
    } else if constexpr (EPI == EPI_STORE_TMA) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 32; i += 2) w[i >> 1] = pack_bf16x2(v[i], v[i + 1]);
      store_block(w, col0, m0 + q * 32);
    } else if constexpr (EPI == EPI_STORE_BF16) {
      if (row_ok) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) w[i >> 1] = pack_bf16x2(v[i], v[i + 1]);
        uint16_t* dst = p.out_bf16 + (int64_t)grow * p.ld_bf16 + col0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (8 * k < nvalid) st_global_v4(dst + 8 * k, w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
      }
    } else {  // EPI_F32
      if (row_ok) {
        float* dst = p.out_f32 + out_off + (int64_t)grow * p.ld_f32 + col0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (4 * k >= nvalid) break;
          float4 x = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
          if (p.f32_mode != F32_STORE) {
            const float4 o = *reinterpret_cast<const float4*>(dst + 4 * k);
            x.x += o.x; x.y += o.y; x.z += o.z; x.w += o.w;
          }
          if (p.f32_mode == F32_ADD_TO_BF16) {
            uint16_t* d16 = p.out_bf16 + (int64_t)grow * p.ld_bf16 + col0 + 4 * k;
            *reinterpret_cast<uint2*>(d16) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
          } else {
            *reinterpret_cast<float4*>(dst + 4 * k) = x;
          }
        }
      }
    }
  };

  for (int j = 0; j < ntiles; ++j) {
    const int acc = NBUF == 2 ? ((tile_base + j) & 1) : 0;
    const uint32_t acc_phase = NBUF == 2 ? ((uint32_t)((tile_base + j) >> 1) & 1u) : ((uint32_t)(tile_base + j) & 1u);
    if constexpr (EPI == EPI_F32) {
      // Pull this row's slice of the fp32 accumulator into L2 while the MMAs run, so the
      // read-modify-write below hits L2.
      if (row_ok && p.f32_mode != F32_STORE) {
#pragma unroll
        for (int sg = 0; sg < kSegs; ++sg) {
          const int n0p = (t_begin + j) * TILE_N + (SPLIT ? sg * (TILE_N / 2) + group * kSegCols : c_lo);
          const int ncols = min(kSegCols, p.N - n0p);
          if (ncols > 0)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.out_f32 + out_off + (int64_t)grow * p.ld_f32 + n0p),
                         "r"((uint32_t)ncols * 4u)
                         : "memory");
        }
      }
    }
    if constexpr (!SPLIT) {
      if (!mbar_wait(acc_full[acc], acc_phase, abort_v, p.err, kErrTimeoutEpilogue)) {
        ok = false;
        break;
      }
      tc_fence_after();
    }
    const int n0 = (t_begin + j) * TILE_N;
    const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * TILE_N);
    if constexpr (SPLIT) {
      // Each half has its own full barrier (the MMA issuer finishes the first half of a tile
      // before the second): wait for the half, load its columns, release it, then compute from
      // registers.
      bool waited = true;
#pragma unroll
      for (int sg = 0; sg < 2; ++sg) {
        if (!mbar_wait(acc_full[sg], acc_phase, abort_v, p.err, kErrTimeoutEpilogue)) {
          waited = false;
          break;
        }
        tc_fence_after();
        const int cs = sg * (TILE_N / 2) + group * kSegCols;
        float v[kSegCols];
#pragma unroll
        for (int cc = 0; cc < kSegCols; cc += 32) tmem_ld32p(tbase + (uint32_t)(cs + cc), v + cc);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc_empty[sg]);
#pragma unroll
        for (int cc = 0; cc < kSegCols; cc += 32)
          if (n0 + cs + cc < p.N) chunk(v + cc, n0 + cs + cc);
      }
      if (!waited) {
        ok = false;
        break;
      }
    } else {
#pragma unroll 1
      for (int c = c_lo; c < c_lo + kCols; c += 32) {
        const int col0 = n0 + c;
        if (col0 >= p.N) break;  // warp-uniform
        float v[32];
        tmem_ld32p(tbase + (uint32_t)c, v);
        tmem_wait_ld();
        chunk(v, col0);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (cluster_arrive) mbar_arrive_cluster(acc_empty[acc]);
        else mbar_arrive(acc_empty[acc]);
      }
    }
  }
  if constexpr (EPI == EPI_STORE_TMA) {
    // The staging tiles are free for the next unit; the kernel waits for the stores themselves.
    if (lane == 0) bulk_wait_read_all();
    __syncwarp();
  } else if constexpr (is_staged(EPI)) {
    // Every TMA store of this warp has completed before the CTA can exit.
    if (stage_smem != 0 && lane == 0) bulk_wait_all();
    __syncwarp();
  }
  if constexpr (is_lse(EPI)) {
    if (row_ok && !*abort_v) {
      const int set = split * GROUPS + group;
      p.part_m[(int64_t)set * p.M + grow] = run_m;
      p.part_s[(int64_t)set * p.M + grow] = run_s;
      if (found) p.part_t[grow] = tval;
    }
  }
  if constexpr (is_tail(EPI)) {
    if (row_ok && !*abort_v) {
      const int64_t o = (int64_t)(split * GROUPS + group) * p.M + grow;
      p.part_m[o] = run_m;
      p.part_s[o] = run_s;
      if (p.part_x != nullptr) p.part_x[o] = sum_x;
      if (p.part_c != nullptr) p.part_c[o] = run_c;
    }
  }
  return ok;
}

template <int EPI, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kThreads, 1)
    lmhead_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages], acc_full[2], acc_empty[2], drain_bar;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;

  const int split = p.split_major ? blockIdx.x : blockIdx.y;
  const int m_blk = p.split_major ? blockIdx.y : blockIdx.x;
  const int m0 = m_blk * BM;
  const int t_begin = split * p.tiles_per_split;
  const int t_end = min(t_begin + p.tiles_per_split, p.n_tiles);
  const int ntiles = t_end - t_begin;
  const int nk = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&acc_full[a]), 1);
      mbar_init(smem_u32(&acc_empty[a]), kEpiWarps);
    }
    mbar_init(smem_u32(&drain_bar), 1);
    abort_flag = 0;
    fence_barrier_init();
    fence_async_shared();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_holder), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_holder;
  volatile int* abort_v = &abort_flag;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0 && ntiles > 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued_phase[kStages];
#pragma unroll
      for (int s = 0; s < kStages; ++s) issued_phase[s] = -1;
      bool ok = true;
      for (int t = t_begin; t < t_end && ok; ++t) {
        const int n0 = t * BN;
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_v, p.err, kErrTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint32_t fb = smem_u32(&full_bar[stage]);
          mbar_arrive_expect_tx(fb, kStageBytes);
          const uint32_t a_dst = smem_base + stage * kStageBytes;
          const uint32_t b_dst = a_dst + kTileA;
          const int k0 = kb * BK;
          if constexpr (!A_MN) {
            tma_load_2d(a_dst, &tmA, fb, k0, m0);
          } else {
#pragma unroll
            for (int c = 0; c < BM / 64; ++c) tma_load_2d(a_dst + c * kMnAtomBytes, &tmA, fb, m0 + 64 * c, k0);
          }
          if constexpr (!B_MN) {
            tma_load_2d(b_dst, &tmB, fb, k0, n0);
          } else {
#pragma unroll
            for (int c = 0; c < BN / 64; ++c) tma_load_2d(b_dst + c * kMnAtomBytes, &tmB, fb, n0 + 64 * c, k0);
          }
          issued_phase[stage] = (int)phase;
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      if (ok) {
        // Tail: wait until the MMA warp has released every stage, so no arrive is pending.
        for (int s = 0; s < kStages; ++s) {
          if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_v, p.err, kErrTimeoutProducer)) break;
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      } else {
        // Abort: let every issued copy land before shared memory is released.
        for (int s = 0; s < kStages; ++s)
          if (issued_phase[s] >= 0) mbar_wait_drain(smem_u32(&full_bar[s]), (uint32_t)issued_phase[s], p.err);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && ntiles > 0) {
      uint32_t idesc = idesc_bf16_f32(BM, BN, A_MN, B_MN);
      if constexpr (takes_f16(EPI)) idesc = p.f16 ? idesc_f16_f32(BM, BN, A_MN, B_MN) : idesc;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int j = 0; j < ntiles && ok; ++j) {
        const int acc = j & 1;
        const uint32_t acc_phase = (uint32_t)(j >> 1) & 1u;
        if (!mbar_wait(smem_u32(&acc_empty[acc]), acc_phase ^ 1u, abort_v, p.err, kErrTimeoutMma)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait(smem_u32(&full_bar[stage]), phase, abort_v, p.err, kErrTimeoutMma)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_base + stage * kStageBytes;
          const uint32_t b_addr = a_addr + kTileA;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t ad = A_MN ? smem_desc(a_addr + k * 2048, kMnAtomBytes, 1024)
                                     : smem_desc(a_addr + k * 32, 16, 1024);
            const uint64_t bd = B_MN ? smem_desc(b_addr + k * 2048, kMnAtomBytes, 1024)
                                     : smem_desc(b_addr + k * 32, 16, 1024);
            mma_bf16(d_tmem, ad, bd, idesc, (kb | k) != 0 ? 1u : 0u);
          }
          mma_commit(smem_u32(&empty_bar[stage]));
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
        if (ok) mma_commit(smem_u32(&acc_full[acc]));
      }
      if (!ok) {
        // Abort: wait for the MMAs already issued before TMEM and shared memory go away.
        mma_commit(smem_u32(&drain_bar));
        mbar_wait_drain(smem_u32(&drain_bar), 0, p.err);
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const uint32_t af[2] = {smem_u32(&acc_full[0]), smem_u32(&acc_full[1])};
    const uint32_t ae[2] = {smem_u32(&acc_empty[0]), smem_u32(&acc_empty[1])};
    epilogue_role<EPI>(p, tmem_base, m0, split, t_begin, t_end, warp, lane, af, ae, false, abort_v);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// CTA-pair variant (cluster of two, tcgen05 cta_group::2): the pair computes a 256 x 256 tile
// per MMA; each CTA stages its own 128 A rows and 128 of the 256 B rows, so shared-memory and
// L2 traffic per MMA flop is 2/3 of the single-CTA kernel and the ring is 6 stages deep.  The
// even CTA issues the MMAs and commits to both CTAs' barriers; both CTAs run the epilogue on
// their own 128 accumulator rows and release the accumulator on the even CTA's barrier.
#ifndef IKRL_PAIR_STAGES
#define IKRL_PAIR_STAGES 6
#endif
constexpr int kPairStages = IKRL_PAIR_STAGES;
constexpr uint32_t kPairTileB = (BN / 2) * BK * 2;  // 16 KB: this CTA's half of the B tile
constexpr uint32_t kPairStageBytes = kTileA + kPairTileB;
constexpr uint32_t kPairSmemBytes = kPairStages * kPairStageBytes + 1024;

// Pacing of the persistent pairs: pairs that read the same W tiles through L2 drift apart over a
// sweep, and a tile read by a leading pair is evicted before the trailing pairs reach it.  Each
// pair publishes how many checkpoints it has passed (one per pace_kb K blocks, default 128: one per
// two tiles at K = 4096, 8 tiles at K = 1024; a long reduction such as dH over the vocabulary has
// many per tile); a pair about to pass checkpoint j waits until every unfinished pair has passed
// checkpoint j - pace_lag (default 1).  The wait is a heuristic with a short bound: after
// kPaceBoundNs without progress the pair stops pacing for the rest of the launch (a pair that is
// not resident, e.g. on a shared GPU, must not stall the others).
constexpr uint64_t kPaceBoundNs = 20000;
constexpr unsigned kPaceDone = 0xffffffffu;

__device__ __forceinline__ unsigned ld_relaxed_u32(const unsigned* ptr) {
  unsigned v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(ptr) : "memory");
  return v;
}
__device__ __forceinline__ void st_relaxed_u32(unsigned* ptr, unsigned v) {
  asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(ptr), "r"(v) : "memory");
}

// Publish "passed checkpoint j" (counted over all of this pair's units) and wait for the laggards.
__device__ __forceinline__ void pace_checkpoint(unsigned* prog, int pair_id, int npairs, int j, int lag,
                                                bool& pacing) {
  st_relaxed_u32(prog + pair_id, (unsigned)j + 1u);
  if (!pacing || j < lag) return;
  const unsigned need = (unsigned)(j + 1 - lag);
  const uint64_t t0 = globaltimer();
  while (true) {
    unsigned mn = kPaceDone;
    for (int q = 0; q < npairs; q += 8) {
      unsigned v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (q + i < npairs) ? ld_relaxed_u32(prog + q + i) : kPaceDone;
#pragma unroll
      for (int i = 0; i < 8; ++i) mn = min(mn, v[i]);
    }
    if (mn >= need) return;
    if (globaltimer() - t0 > kPaceBoundNs) {
      pacing = false;
      return;
    }
    __nanosleep(256);
  }
}

template <int EPI, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kThreads, 1)
    lmhead_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                            const __grid_constant__ CUtensorMap tmC, const GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kPairStages], empty_bar[kPairStages], acc_full[2], acc_empty[2], drain_bar;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t rank = cluster_ctarank();

  // Persistent pairs.  A work unit is (split, row-block pair); unit u covers split u % splits and
  // row blocks 2 * (u / splits) + {0, 1}.  Pair c processes units c, c + npairs, ...; the units
  // in flight at any time are consecutive, so pairs that run together share the B tiles of a
  // split and the A rows of a row-block pair through L2, and proceed in step.
  const int pair_id = blockIdx.x >> 1;
  const int npairs = gridDim.x >> 1;
  const int m_pairs = (((live_rows<EPI>(p) + BM - 1) / BM) + 1) >> 1;
  const int splits = column_splits<EPI>(p), tps = split_tiles<EPI>(p);
  const int nunits = m_pairs * splits;
  const int nk = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&acc_full[a]), 1);
      mbar_init(smem_u32(&acc_empty[a]), 2 * kEpiWarps);
    }
    mbar_init(smem_u32(&drain_bar), 1);
    abort_flag = 0;
    fence_barrier_init();
    fence_async_shared();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&tmem_holder), kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers initialised and TMEM allocated before any cross-CTA use
  tc_fence_after();
  const uint32_t tmem_base = tmem_holder;
  volatile int* abort_v = &abort_flag;

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      bool pacing = p.lockstep != nullptr && rank == 0;
      const uint64_t pol_a = l2_policy(p.a_policy);
      const uint64_t pol_b = l2_policy(p.b_policy);
      int jt = 0;
      for (int u = pair_id; u < nunits && ok; u += npairs) {
        const int split = u % splits;
        const int m0 = (2 * (u / splits) + (int)rank) * BM;
        const int t_begin = split * tps;
        const int t_end = min(t_begin + tps, p.n_tiles);
        for (int t = t_begin; t < t_end && ok; ++t, ++jt) {
          const int nb = t * BN + (int)rank * (BN / 2);  // this CTA's half of the N tile
          for (int kb = 0; kb < nk; ++kb) {
            const int gkb = jt * nk + kb;
            if (p.lockstep != nullptr && rank == 0 && gkb % p.pace_kb == 0)
              pace_checkpoint(p.lockstep, pair_id, npairs, gkb / p.pace_kb, p.pace_lag, pacing);
            if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_v, p.err, kErrTimeoutProducer)) {
              ok = false;
              break;
            }
            const uint32_t fb_local = smem_u32(&full_bar[stage]);
            const uint32_t fb_leader = mapa_shared(fb_local, 0);
            if (rank == 0) mbar_arrive_expect_tx(fb_local, 2 * kPairStageBytes);
            const uint32_t a_dst = smem_base + stage * kPairStageBytes;
            const uint32_t b_dst = a_dst + kTileA;
            const int k0 = kb * BK;
            if constexpr (!A_MN) {
              tma_load_2d_pair_hint(a_dst, &tmA, fb_leader, k0, m0, pol_a);
            } else {
#pragma unroll
              for (int c = 0; c < BM / 64; ++c)
                tma_load_2d_pair_hint(a_dst + c * kMnAtomBytes, &tmA, fb_leader, m0 + 64 * c, k0, pol_a);
            }
            if constexpr (!B_MN) {
              tma_load_2d_pair_hint(b_dst, &tmB, fb_leader, k0, nb, pol_b);
            } else {
#pragma unroll
              for (int c = 0; c < BN / 128; ++c)
                tma_load_2d_pair_hint(b_dst + c * kMnAtomBytes, &tmB, fb_leader, nb + 64 * c, k0, pol_b);
            }
            if (++stage == kPairStages) { stage = 0; phase ^= 1u; }
          }
        }
      }
      if (p.lockstep != nullptr && rank == 0) st_relaxed_u32(p.lockstep + pair_id, kPaceDone);
      if (ok) {
        for (int s = 0; s < kPairStages; ++s) {
          if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_v, p.err, kErrTimeoutProducer)) break;
          if (++stage == kPairStages) { stage = 0; phase ^= 1u; }
        }
      } else {
        // Abort: the copies' completion is counted on the even CTA's barrier, which this CTA
        // cannot wait on; give copies already issued 1 ms to land before shared memory goes away.
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (even CTA only) ----------------
    if (rank == 0 && lane == 0) {
      uint32_t idesc = idesc_bf16_f32(2 * BM, BN, A_MN, B_MN);
      if constexpr (takes_f16(EPI)) idesc = p.f16 ? idesc_f16_f32(2 * BM, BN, A_MN, B_MN) : idesc;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int j = 0;  // tiles issued so far (accumulator ring position)
      for (int u = pair_id; u < nunits && ok; u += npairs) {
        const int split = u % splits;
        const int t_begin = split * tps;
        const int t_end = min(t_begin + tps, p.n_tiles);
        for (int t = t_begin; t < t_end && ok; ++t, ++j) {
          const int acc = j & 1;
          const uint32_t acc_phase = (uint32_t)(j >> 1) & 1u;
          if (!mbar_wait(smem_u32(&acc_empty[acc]), acc_phase ^ 1u, abort_v, p.err, kErrTimeoutMma)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
          for (int kb = 0; kb < nk; ++kb) {
            if (!mbar_wait(smem_u32(&full_bar[stage]), phase, abort_v, p.err, kErrTimeoutMma)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a_addr = smem_base + stage * kPairStageBytes;
            const uint32_t b_addr = a_addr + kTileA;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              const uint64_t ad = A_MN ? smem_desc(a_addr + k * 2048, kMnAtomBytes, 1024)
                                       : smem_desc(a_addr + k * 32, 16, 1024);
              const uint64_t bd = B_MN ? smem_desc(b_addr + k * 2048, kMnAtomBytes, 1024)
                                       : smem_desc(b_addr + k * 32, 16, 1024);
              mma_bf16_pair(d_tmem, ad, bd, idesc, (kb | k) != 0 ? 1u : 0u);
            }
            const uint32_t eb = smem_u32(&empty_bar[stage]);
            mma_commit_pair(mapa_shared(eb, 0));
            mma_commit_pair(mapa_shared(eb, 1));
            if (++stage == kPairStages) { stage = 0; phase ^= 1u; }
          }
          if (ok) {
            const uint32_t fb = smem_u32(&acc_full[acc]);
            mma_commit_pair(mapa_shared(fb, 0));
            mma_commit_pair(mapa_shared(fb, 1));
          }
        }
      }
      if (!ok) {
        mma_commit_pair(mapa_shared(smem_u32(&drain_bar), 0));
        mbar_wait_drain(smem_u32(&drain_bar), 0, p.err);
      }
    }
  } else {
    // ---------------- epilogue (both CTAs, own 128 rows) ----------------
    const uint32_t af[2] = {smem_u32(&acc_full[0]), smem_u32(&acc_full[1])};
    const uint32_t ae[2] = {mapa_shared(smem_u32(&acc_empty[0]), 0), mapa_shared(smem_u32(&acc_empty[1]), 0)};
    int jb = 0;
    for (int u = pair_id; u < nunits; u += npairs) {
      const int split = u % splits;
      const int m0 = (2 * (u / splits) + (int)rank) * BM;
      const int t_begin = split * tps;
      const int t_end = min(t_begin + tps, p.n_tiles);
      if (!epilogue_role<EPI>(p, tmem_base, m0, split, t_begin, t_end, warp, lane, af, ae, true, abort_v, jb)) break;
      jb += t_end - t_begin;
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still touch its barriers or shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// Wide CTA-pair variant for long K: the pair computes a 256 x 512 tile per K step with two
// N=256 MMAs into all 512 TMEM columns.  Each CTA stages 128 A rows and 256 of the 512 B rows per
// 64-deep K block (48 KB, 4 stages), so L2 and shared-memory reads per MMA flop are 3/4 of the
// 256 x 256 pair kernel.  The single accumulator is not double-buffered; it is drained in two
// 256-column halves, and the next tile's first-half MMAs start as soon as the first half is
// drained, so only that half's drain delays the tensor pipe.
constexpr int WN = 512;
constexpr int kWideStages = 4;
constexpr uint32_t kWideTileB = (WN / 2) * BK * 2;  // 32 KB: this CTA's half of the B tile
constexpr uint32_t kWideStageBytes = kTileA + kWideTileB;
constexpr uint32_t kWideSmemBytes = kWideStages * kWideStageBytes + 1024;
// DLOGITS adds one 32 x 32 bf16 staging tile per epilogue warp for the TMA stores of dS.
constexpr uint32_t kWideDsSmemBytes = kWideSmemBytes + kWideEpiWarps * kDsStageBytes;
static_assert(kWideDsSmemBytes <= 232448 - 256, "wide DLOGITS kernel exceeds the shared memory of a CTA");

template <int EPI, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kWideThreads, 1)
    lmhead_gemm_wide_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                            const __grid_constant__ CUtensorMap tmC, const GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kWideStages], empty_bar[kWideStages], acc_full[2], acc_empty[2], drain_bar;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t rank = cluster_ctarank();
  const int pair_id = blockIdx.x >> 1;
  const int npairs = gridDim.x >> 1;
  const int m_pairs = (((live_rows<EPI>(p) + BM - 1) / BM) + 1) >> 1;
  const int kspl = p.ksplits > 1 ? p.ksplits : 1;
  const int splits = column_splits<EPI>(p), tps = split_tiles<EPI>(p);
  const int nunits = m_pairs * splits * kspl;
  const int nk_all = (p.K + BK - 1) / BK;
  // Work unit u: K range ks (slowest, so the units in flight share it), then the row pair, then
  // the vocab split (fastest), as without K ranges.
  auto unit_of = [&](int u, int& mp, int& split, int& ks, int& kb0, int& kb1) {
    const int per = m_pairs * splits;
    ks = u / per;
    const int r = u - ks * per;
    split = r % splits;
    mp = r / splits;
    kb0 = (int)((int64_t)ks * nk_all / kspl);
    kb1 = (int)((int64_t)(ks + 1) * nk_all / kspl);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kWideStages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&acc_full[a]), 1);
      mbar_init(smem_u32(&acc_empty[a]), 2 * kWideEpiWarps);
    }
    mbar_init(smem_u32(&drain_bar), 1);
    abort_flag = 0;
    fence_barrier_init();
    fence_async_shared();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&tmem_holder), kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = tmem_holder;
  volatile int* abort_v = &abort_flag;

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    if (lane == 0) {
      const uint64_t pol_a = l2_policy(p.a_policy);
      const uint64_t pol_b = l2_policy(p.b_policy);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      bool pacing = p.lockstep != nullptr && rank == 0;
      int gkb = 0;  // K blocks this pair has loaded
      for (int u = pair_id; u < nunits && ok; u += npairs) {
        int mp, split, ks, kb0, kb1;
        unit_of(u, mp, split, ks, kb0, kb1);
        const int m0 = (2 * mp + (int)rank) * BM;
        const int t_begin = split * tps;
        const int t_end = min(t_begin + tps, p.n_tiles);
        for (int t = t_begin; t < t_end && ok; ++t) {
          for (int kb = kb0; kb < kb1; ++kb, ++gkb) {
            // pacing checkpoint every pace_kb K blocks of this pair's work
            if (p.lockstep != nullptr && rank == 0 && gkb % p.pace_kb == 0)
              pace_checkpoint(p.lockstep, pair_id, npairs, gkb / p.pace_kb, p.pace_lag, pacing);
            if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_v, p.err, kErrTimeoutProducer)) {
              ok = false;
              break;
            }
            const uint32_t fb_local = smem_u32(&full_bar[stage]);
            const uint32_t fb_leader = mapa_shared(fb_local, 0);
            if (rank == 0) mbar_arrive_expect_tx(fb_local, 2 * kWideStageBytes);
            const uint32_t a_dst = smem_base + stage * kWideStageBytes;
            const uint32_t b_dst = a_dst + kTileA;
            const int k0 = kb * BK;
            if constexpr (!A_MN) {
              tma_load_2d_pair_hint(a_dst, &tmA, fb_leader, k0, m0, pol_a);
            } else {
#pragma unroll
              for (int c = 0; c < BM / 64; ++c)
                tma_load_2d_pair_hint(a_dst + c * kMnAtomBytes, &tmA, fb_leader, m0 + 64 * c, k0, pol_a);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // B rows of MMA h that this CTA provides: [t*512 + 256h + 128*rank, +128)
              const int nb = t * WN + h * BN + (int)rank * (BN / 2);
              const uint32_t bh = b_dst + h * ((BN / 2) * BK * 2);
              if constexpr (!B_MN) {
                tma_load_2d_pair_hint(bh, &tmB, fb_leader, k0, nb, pol_b);
              } else {
#pragma unroll
                for (int c = 0; c < BN / 128; ++c)
                  tma_load_2d_pair_hint(bh + c * kMnAtomBytes, &tmB, fb_leader, nb + 64 * c, k0, pol_b);
              }
            }
            if (++stage == kWideStages) { stage = 0; phase ^= 1u; }
          }
        }
      }
      if (p.lockstep != nullptr && rank == 0) st_relaxed_u32(p.lockstep + pair_id, kPaceDone);
      if (ok) {
        for (int s = 0; s < kWideStages; ++s) {
          if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_v, p.err, kErrTimeoutProducer)) break;
          if (++stage == kWideStages) { stage = 0; phase ^= 1u; }
        }
      } else {
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (even CTA only) ----------------
    if (rank == 0 && lane == 0) {
      uint32_t idesc = idesc_bf16_f32(2 * BM, BN, A_MN, B_MN);
      if constexpr (takes_f16(EPI)) idesc = p.f16 ? idesc_f16_f32(2 * BM, BN, A_MN, B_MN) : idesc;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int j = 0;
      for (int u = pair_id; u < nunits && ok; u += npairs) {
        int mp, split, ks, kb0, kb1;
        unit_of(u, mp, split, ks, kb0, kb1);
        const int nk = kb1 - kb0;  // K blocks of this unit; kb below counts from its first
        const int t_begin = split * tps;
        const int t_end = min(t_begin + tps, p.n_tiles);
        // MMAs of one K block into accumulator half h (TMEM columns [256h, 256h + 256)).
        auto issue_half = [&](int st, int kb, int h) {
          const uint32_t a_addr = smem_base + st * kWideStageBytes;
          const uint32_t bh = a_addr + kTileA + h * ((BN / 2) * BK * 2);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t ad = A_MN ? smem_desc(a_addr + k * 2048, kMnAtomBytes, 1024)
                                     : smem_desc(a_addr + k * 32, 16, 1024);
            const uint64_t bd = B_MN ? smem_desc(bh + k * 2048, kMnAtomBytes, 1024) : smem_desc(bh + k * 32, 16, 1024);
            mma_bf16_pair(tmem_base + (uint32_t)(h * BN), ad, bd, idesc, (kb | k) != 0 ? 1u : 0u);
          }
        };
        auto release_stage = [&](int st) {
          const uint32_t eb = smem_u32(&empty_bar[st]);
          mma_commit_pair(mapa_shared(eb, 0));
          mma_commit_pair(mapa_shared(eb, 1));
        };
        for (int t = t_begin; t < t_end && ok; ++t, ++j) {
          const uint32_t epar = ((uint32_t)j & 1u) ^ 1u;
          if (!mbar_wait(smem_u32(&acc_empty[0]), epar, abort_v, p.err, kErrTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          // The first half of the accumulator is free: run its MMAs over the K blocks already
          // staged while the epilogue still drains the second half.
          const int look = min(kWideStages, nk);
          {
            int st = stage;
            uint32_t ph = phase;
            for (int kb = 0; kb < look; ++kb) {
              if (!mbar_wait(smem_u32(&full_bar[st]), ph, abort_v, p.err, kErrTimeoutMma)) { ok = false; break; }
              tc_fence_after();
              issue_half(st, kb, 0);
              if (++st == kWideStages) { st = 0; ph ^= 1u; }
            }
          }
          if (!ok) break;
          auto commit_full = [&](int h) {
            const uint32_t fb = smem_u32(&acc_full[h]);
            mma_commit_pair(mapa_shared(fb, 0));
            mma_commit_pair(mapa_shared(fb, 1));
          };
          if (look == nk) commit_full(0);  // the whole first half is issued
          if (!mbar_wait(smem_u32(&acc_empty[1]), epar, abort_v, p.err, kErrTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          for (int kb = 0; kb < look; ++kb) {
            issue_half(stage, kb, 1);
            release_stage(stage);
            if (++stage == kWideStages) { stage = 0; phase ^= 1u; }
          }
          // The last `tail` K blocks run first-half-first: the first half is final while the
          // second half's last MMAs still run, so the epilogue drains it and releases it for the
          // next tile without idling the tensor pipe.
          const int tail = min(min(p.split_tail, kWideStages), nk - look);
          for (int kb = look; kb < nk - tail; ++kb) {
            if (!mbar_wait(smem_u32(&full_bar[stage]), phase, abort_v, p.err, kErrTimeoutMma)) { ok = false; break; }
            tc_fence_after();
            issue_half(stage, kb, 0);
            issue_half(stage, kb, 1);
            release_stage(stage);
            if (++stage == kWideStages) { stage = 0; phase ^= 1u; }
          }
          if (!ok) break;
          if (tail > 0) {
            int st = stage;
            uint32_t ph = phase;
            for (int kb = nk - tail; kb < nk; ++kb) {
              if (!mbar_wait(smem_u32(&full_bar[st]), ph, abort_v, p.err, kErrTimeoutMma)) { ok = false; break; }
              tc_fence_after();
              issue_half(st, kb, 0);
              if (++st == kWideStages) { st = 0; ph ^= 1u; }
            }
            if (!ok) break;
            commit_full(0);
            for (int kb = nk - tail; kb < nk; ++kb) {
              issue_half(stage, kb, 1);
              release_stage(stage);
              if (++stage == kWideStages) { stage = 0; phase ^= 1u; }
            }
          } else if (look < nk) {
            commit_full(0);
          }
          commit_full(1);
        }
      }
      if (!ok) {
        mma_commit_pair(mapa_shared(smem_u32(&drain_bar), 0));
        mbar_wait_drain(smem_u32(&drain_bar), 0, p.err);
      }
    }
  } else {
    // ---------------- epilogue (both CTAs, own 128 rows x 512 columns) ----------------
    const uint32_t af[2] = {smem_u32(&acc_full[0]), smem_u32(&acc_full[1])};
    const uint32_t ae[2] = {mapa_shared(smem_u32(&acc_empty[0]), 0), mapa_shared(smem_u32(&acc_empty[1]), 0)};
    const uint32_t stage = (is_staged(EPI) && p.ds_tma)
                               ? smem_base + kWideStages * kWideStageBytes + (uint32_t)(warp - 2) * kDsStageBytes
                               : 0u;
    int jb = 0;
    for (int u = pair_id; u < nunits; u += npairs) {
      int mp, split, ks, kb0, kb1;
      unit_of(u, mp, split, ks, kb0, kb1);
      const int m0 = (2 * mp + (int)rank) * BM;
      const int t_begin = split * tps;
      const int t_end = min(t_begin + tps, p.n_tiles);
      if (!epilogue_role<EPI, WN, 1, kWideGroups, true>(p, tmem_base, m0, split, t_begin, t_end, warp, lane, af, ae,
                                                        true, abort_v, jb, &tmC, stage, (int64_t)ks * p.ks_stride))
        break;
      jb += t_end - t_begin;
    }
    if constexpr (EPI == EPI_STORE_TMA) {
      if (lane == 0) bulk_wait_all();
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// Merge the per-split (max, sum) pairs of each row: lse = ln2 * (M + log2 sum_s s_s 2^(m_s - M)).
__global__ void lse_combine_kernel(const float* __restrict__ part_m, const float* __restrict__ part_s,
                                   const float* __restrict__ part_t, const int64_t* __restrict__ ids, int M,
                                   int V, int splits, float* __restrict__ logp, float* __restrict__ lse_out,
                                   const int* __restrict__ err) {
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= M) return;
  const bool bad = *err != 0;
  float mx = -INFINITY;
  for (int s = 0; s < splits; ++s) mx = fmaxf(mx, part_m[(int64_t)s * M + r]);
  float sum = 0.f;
  for (int s = 0; s < splits; ++s) sum += part_s[(int64_t)s * M + r] * fast_exp2(part_m[(int64_t)s * M + r] - mx);
  const float lse = (mx + log2f(sum)) * kLn2;
  const int64_t t = ids[r];
  float lp;
  if (bad) lp = __int_as_float(0x7fc00000);
  else if (t == -100) lp = -0.f;
  else if (t < 0 || t >= V) lp = __int_as_float(0x7fc00000);
  else lp = part_t[r] - lse;
  logp[r] = lp;
  if (lse_out) lse_out[r] = bad ? __int_as_float(0x7fc00000) : lse;
}

// Vocab shard of the forward: the shard's own logsumexp and the raw target logit when the target
// id falls in this shard (-inf otherwise, so that a max over shards picks the owner's value).
__global__ void lse_shard_combine_kernel(const float* __restrict__ part_m, const float* __restrict__ part_s,
                                         const float* __restrict__ part_t, const int64_t* __restrict__ ids, int M,
                                         int64_t vocab_start, int V_shard, int splits, float* __restrict__ tlogit,
                                         float* __restrict__ lse_out, const int* __restrict__ err) {
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= M) return;
  const bool bad = *err != 0;
  float mx = -INFINITY;
  for (int s = 0; s < splits; ++s) mx = fmaxf(mx, part_m[(int64_t)s * M + r]);
  float sum = 0.f;
  for (int s = 0; s < splits; ++s) sum += part_s[(int64_t)s * M + r] * fast_exp2(part_m[(int64_t)s * M + r] - mx);
  const float nan = __int_as_float(0x7fc00000);
  lse_out[r] = bad ? nan : (mx + log2f(sum)) * kLn2;
  const int64_t t = ids[r];
  const bool owned = t != -100 && t >= vocab_start && t < vocab_start + V_shard;
  tlogit[r] = bad ? nan : (owned ? part_t[r] : -INFINITY);
}

// log p = t - logsumexp over shards, from each shard's (target logit or -inf, shard logsumexp):
// parts[q][0][r], parts[q][1][r] for shards q < P.  Ignored rows give -0.0 and ids outside the
// vocabulary NaN, as the unsharded forward.
__global__ void vocab_parallel_combine_kernel(const float* __restrict__ parts, const int64_t* __restrict__ ids,
                                              int64_t N, int P, int64_t V_total, float* __restrict__ logp,
                                              float* __restrict__ lse_out) {
  const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= N) return;
  float mx = -INFINITY, t = -INFINITY;
  bool nan_in = false;
  for (int q = 0; q < P; ++q) {
    const float lq = parts[((int64_t)q * 2 + 1) * N + r];
    const float tq = parts[((int64_t)q * 2) * N + r];
    nan_in |= (lq != lq) || (tq != tq);
    mx = fmaxf(mx, lq);
    t = fmaxf(t, tq);
  }
  float sum = 0.f;
  for (int q = 0; q < P; ++q) sum += expf(parts[((int64_t)q * 2 + 1) * N + r] - mx);
  const float nan = __int_as_float(0x7fc00000);
  const float lse = nan_in ? nan : mx + logf(sum);
  const int64_t id = ids[r];
  float lp;
  if (id == -100) lp = -0.f;
  else if (id < 0 || id >= V_total) lp = nan;
  else lp = t - lse;
  logp[r] = lp;
  if (lse_out) lse_out[r] = lse;
}

// ---- host side ---------------------------------------------------------------------------------

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// 2-D bf16 tensor map over a row-major matrix [outer, inner] with row stride `ld` elements and a
// box of {64 inner, box_outer} elements, 128-byte swizzle, zero fill out of bounds.
int make_tmap(CUtensorMap* m, const void* base, uint64_t inner, uint64_t outer, uint64_t ld, uint32_t box_outer,
              const char* what) {
  EncodeTiledFn fn = encode_fn();
  IKRL_REQUIRE(fn != nullptr, IKRL_ERR_CUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(base) & 15) == 0, IKRL_ERR_ALIGNMENT,
               "%s: base address must be 16-byte aligned", what);
  IKRL_REQUIRE((ld * 2) % 16 == 0, IKRL_ERR_ALIGNMENT, "%s: row stride %llu elements is not a multiple of 8", what,
               (unsigned long long)ld);
  const cuuint64_t dims[2] = {inner, outer};
  const cuuint64_t strides[1] = {ld * 2};
  const cuuint32_t box[2] = {64, box_outer};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  IKRL_REQUIRE(r == CUDA_SUCCESS, IKRL_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return IKRL_OK;
}

// Tensor map for the wide kernel's TMA stores of dS: bf16 [outer, inner] with row stride `ld`
// elements, 32 x 32 boxes (64-byte rows) in the 64-byte swizzled shared-memory layout.  Stores clip
// at the inner and outer extents.
int make_store_tmap(CUtensorMap* m, void* base, uint64_t inner, uint64_t outer, uint64_t ld, const char* what) {
  EncodeTiledFn fn = encode_fn();
  IKRL_REQUIRE(fn != nullptr, IKRL_ERR_CUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(base) & 15) == 0, IKRL_ERR_ALIGNMENT,
               "%s: base address must be 16-byte aligned", what);
  IKRL_REQUIRE((ld * 2) % 16 == 0, IKRL_ERR_ALIGNMENT, "%s: row stride %llu elements is not a multiple of 8", what,
               (unsigned long long)ld);
  const cuuint64_t dims[2] = {inner, outer};
  const cuuint64_t strides[1] = {ld * 2};
  const cuuint32_t box[2] = {32, 32};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  IKRL_REQUIRE(r == CUDA_SUCCESS, IKRL_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return IKRL_OK;
}

template <int EPI, bool A_MN, bool B_MN>
int launch_gemm(const CUtensorMap& a, const CUtensorMap& b, const GemmParams& p, int m_tiles, cudaStream_t s) {
  auto kern = lmhead_gemm_kernel<EPI, A_MN, B_MN>;
  IKRL_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes));
  IKRL_REQUIRE(m_tiles <= 65535 || p.split_major == 0, IKRL_ERR_UNSUPPORTED, "too many row blocks (%d)", m_tiles);
  const dim3 grid = p.split_major ? dim3(p.splits, m_tiles) : dim3(m_tiles, p.splits);
  kern<<<grid, kThreads, kSmemBytes, s>>>(a, b, p);
  return check_launch("lmhead_gemm_kernel");
}

// Pair launch: a persistent 1-D grid of one CTA pair (cluster of 2) per two SMs.
// Per-pair tile counters of the pacing in the wide kernel: one array per device, zeroed before
// every launch that paces (launches on one stream are ordered; concurrent launches on other
// streams would share it, which only weakens the pacing, whose waits are bounded).
constexpr int kMaxPacedPairs = 512;
static __device__ unsigned g_pace[kMaxPacedPairs];
std::mutex g_pace_mu;
unsigned* g_pace_addr[64] = {nullptr};

int pace_array(unsigned** out) {
  int dev = 0;
  IKRL_CUDA(cudaGetDevice(&dev));
  IKRL_REQUIRE(dev >= 0 && dev < 64, IKRL_ERR_UNSUPPORTED, "device ordinal %d out of range", dev);
  std::lock_guard<std::mutex> lock(g_pace_mu);
  if (g_pace_addr[dev] == nullptr) {
    void* ptr = nullptr;
    IKRL_CUDA(cudaGetSymbolAddress(&ptr, g_pace));
    g_pace_addr[dev] = reinterpret_cast<unsigned*>(ptr);
  }
  *out = g_pace_addr[dev];
  return IKRL_OK;
}

// Pacing of the wide kernel's pairs: IKRL_TUNE_PACE is a mask over the epilogues, bit EPI set =
// launches with that epilogue are paced.  The default (-1) paces every launch except a forward
// with K < 2048: there W is a quarter of the 8B head's bytes, the forward reads little DRAM
// unpaced, and its 16-K-block tiles make the checkpoint waits a larger share.
bool pacing_enabled(int epi, int K) {
  int64_t mask = tuning(IKRL_TUNE_PACE);
  if (mask < 0) mask = K >= 2048 ? 15 : 14;
  return (mask >> epi_kind(epi)) & 1;
}
bool persistent_pairs() { return tuning(IKRL_TUNE_PERSISTENT) != 0; }

template <int EPI, bool A_MN, bool B_MN, bool WIDE>
int launch_gemm_pair(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap* c, const GemmParams& p_in,
                     int m_tiles, cudaStream_t s) {
  GemmParams p = p_in;
  const auto kern = [] {
    if constexpr (WIDE) return lmhead_gemm_wide_kernel<EPI, A_MN, B_MN>;
    else return lmhead_gemm_pair_kernel<EPI, A_MN, B_MN>;
  }();
  p.ds_tma = (WIDE && c != nullptr && is_staged(EPI)) ? 1 : 0;
  const uint32_t smem_bytes = WIDE ? (p.ds_tma ? kWideDsSmemBytes : kWideSmemBytes) : kPairSmemBytes;
  IKRL_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes));
  IKRL_REQUIRE(p.split_major == 1, IKRL_ERR_UNSUPPORTED, "pair kernel needs a split-major grid");
  IKRL_REQUIRE(WIDE || p.ksplits <= 1, IKRL_ERR_UNSUPPORTED, "K ranges need the 256x512 kernel");
  IKRL_REQUIRE(p.ksplits <= 1 || (EPI == EPI_F32 && p.f32_mode == F32_STORE), IKRL_ERR_UNSUPPORTED,
               "K ranges need fp32 partial stores");
  const int64_t nunits = (int64_t)((m_tiles + 1) / 2) * p.splits * std::max(1, p.ksplits);
  IKRL_REQUIRE(nunits <= 0x3fffffffLL, IKRL_ERR_UNSUPPORTED, "too many work units (%lld)", (long long)nunits);
  int dev = 0, nsm = kNumSMs;
  IKRL_CUDA(cudaGetDevice(&dev));
  IKRL_CUDA(cudaDeviceGetAttribute(&nsm, cudaDevAttrMultiProcessorCount, dev));
  // One resident pair per two SMs; IKRL_TUNE_PERSISTENT = 0 launches one pair per unit instead.
  const bool persistent = persistent_pairs();
  const int64_t npairs = std::max<int64_t>(1, persistent ? std::min<int64_t>(nunits, nsm / 2) : nunits);
  p.lockstep = nullptr;
  p.split_tail = (int)tuning(IKRL_TUNE_SPLIT_TAIL);
  // Pacing helps the wide kernel (long tiles, W re-read across pairs); on the 256 x 256 pair
  // kernel at K = 1024 it measured 7% slower (checkpoints every 4 short tiles stall the producer).
  if (WIDE && persistent && npairs <= kMaxPacedPairs && pacing_enabled(EPI, p.K)) {
    int rc = pace_array(&p.lockstep);
    if (rc) return rc;
    IKRL_CUDA(cudaMemsetAsync(p.lockstep, 0, sizeof(unsigned) * (size_t)npairs, s));
    p.pace_kb = (int)tuning((EPI == EPI_F32 || epi_kind(EPI) == EPI_STORE_BF16) ? IKRL_TUNE_PACE_KB_LONG : IKRL_TUNE_PACE_KB);
    p.pace_lag = (int)tuning(IKRL_TUNE_PACE_LAG);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * npairs), 1, 1);
  cfg.blockDim = dim3(WIDE ? kWideThreads : kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, b, p.ds_tma ? *c : a, p);
  if (e != cudaSuccess) {
    int nclusters = -1;
    cudaError_t e2 = cudaOccupancyMaxActiveClusters(&nclusters, kern, &cfg);
    cudaFuncAttributes fa{};
    cudaFuncGetAttributes(&fa, kern);
    (void)cudaGetLastError();
    set_error("pair kernel launch failed: %s (grid %u x %u, max active clusters %d [%s], static smem %zu, "
              "dynamic %u, max dyn %d, regs %d, max threads %d)",
              cudaGetErrorString(e), cfg.gridDim.x, cfg.gridDim.y, nclusters, cudaGetErrorString(e2), fa.sharedSizeBytes,
              smem_bytes, fa.maxDynamicSharedSizeBytes, fa.numRegs, fa.maxThreadsPerBlock);
    return IKRL_ERR_CUDA;
  }
  return check_launch("lmhead_gemm_pair_kernel");
}

// Kernel choice: CTA pairs by default; IKRL_TUNE_CTA_PAIRS = 0 (or ikrl_lmhead_set_cta_pairs(0))
// selects the single-CTA kernel.
bool use_pairs() { return tuning(IKRL_TUNE_CTA_PAIRS) != 0; }

// Wide tiles (256 x 512 per pair) for long reductions: IKRL_TUNE_WIDE 0 never, 1 always, otherwise
// when K >= 1024 (16 K blocks per tile or more; at K = 1024 the Qwen3-0.6B head ran 1.4% faster
// wide than on 256 x 256 pairs).
bool use_wide(int K) {
  const int64_t w = tuning(IKRL_TUNE_WIDE);
  if (w == 0) return false;
  if (w == 1) return true;
  return K >= 1024;
}

int64_t cdiv64(int64_t a, int64_t b);

// Busiest pair's work, in tiles, when m_pairs row pairs x ceil(n_tiles / tps) column ranges of
// tps tiles (the last range shorter) are dealt round-robin, range fastest, to npairs persistent
// pairs: the order of the pair kernels' unit loop.
int64_t pair_makespan(int64_t m_pairs, int n_tiles, int tps, int64_t npairs) {
  const int splits = (int)cdiv64(n_tiles, tps);
  const int64_t nunits = m_pairs * splits;
  const int64_t np = std::max<int64_t>(1, std::min<int64_t>(nunits, npairs));
  int64_t worst = 0;
  for (int64_t pr = 0; pr < np; ++pr) {
    int64_t tiles = 0;
    for (int64_t u = pr; u < nunits; u += np) {
      const int sp = (int)(u % splits);
      tiles += std::min(tps, n_tiles - sp * tps);
    }
    worst = std::max(worst, tiles);
  }
  return worst;
}

// Balance of the persistent pairs: the L2 rule's split count can leave a last round of units on
// a few pairs only (14 m-pairs x 11 splits = 154 units over 74 pairs runs 3 rounds where the mean
// is 2.1).  Up to kBalanceMost times the hinted count, take a larger count when it shortens the busiest
// pair's work by at least 5%; more splits mean more W re-reads, so near-balanced hints stay.  Used for the
// backward's dS launches, which have no per-split workspace, and for the row losses' forward, whose workspace
// holds that many sets (row_loss_fwd_layout; launch_k1 checks it).  IKRL_TUNE_BALANCE_SPLITS = 0 keeps the
// hint.
constexpr int kBalanceMost = 3;
bool balance_splits_enabled() { return tuning(IKRL_TUNE_BALANCE_SPLITS) != 0; }

int balanced_tiles_per_split(int64_t m_tiles, int n_tiles, int splits_hint, int64_t npairs) {
  const int64_t m_pairs = (m_tiles + 1) / 2;
  int best_tps = (int)cdiv64(n_tiles, splits_hint);
  int64_t best = pair_makespan(m_pairs, n_tiles, best_tps, npairs);
  for (int sp = splits_hint + 1; sp <= std::min(kBalanceMost * splits_hint, n_tiles); ++sp) {
    const int tps = (int)cdiv64(n_tiles, sp);
    if (tps == best_tps) continue;
    const int64_t ms = pair_makespan(m_pairs, n_tiles, tps, npairs);
    if (ms * 20 < best * 19) {
      best = ms;
      best_tps = tps;
    }
  }
  return best_tps;
}

// Kernel and column ranges of one K1 GEMM launch: host arithmetic only, no CUDA call.
// kind: 0 single CTAs (128 x 256), 1 CTA pairs (256 x 256), 2 wide CTA pairs (256 x 512).
// splits_hint > 0 asks for that many column ranges (fewer if the tiles run out); splits_hint <= 0
// gives every column tile its own unit.  nsm: SMs of the GPU (one persistent pair per two).
struct K1Plan {
  int kind, n_tiles, tiles_per_split, splits;
};

K1Plan plan_k1(int epi, int64_t m_tiles, int N, int K, int splits_hint, int nsm) {
  K1Plan pl{};
  // A row loss of at most 128 rows takes single CTAs: a pair's MMAs would run 256 rows for it, half of
  // them empty (96 rows x 1024 against 151936 columns: 104 us in 256 x 512 pair tiles, 62 us so).
  pl.kind = !use_pairs() || ((is_tail(epi) || epi == EPI_DTAIL) && m_tiles == 1) ? 0 : (use_wide(K) ? 2 : 1);
  if (epi == EPI_STORE_TMA) pl.kind = 2;
  const bool persistent = persistent_pairs();
  const int64_t npairs = std::max(1, nsm / 2);
  if (epi == EPI_STORE_BF16 && pl.kind == 2 && splits_hint <= 0 && persistent && balance_splits_enabled() &&
      tuning(IKRL_TUNE_WIDE) == -1) {
    // bf16-store launches (dH; a one-chunk bf16 dW): every column tile is a unit reducing over the
    // whole K, so a narrow N leaves few units (dH at H = 1024: 2 wide tiles per row pair; 40 row
    // pairs give 80 units, two rounds on 74 pairs where the mean is 1.08).  256-column tiles halve
    // the unit: take the 256 x 256 pair kernel when its busiest pair finishes at least 5% sooner,
    // counting its measured ~13% lower rate per flop.
    const int64_t m_pairs = (m_tiles + 1) / 2;
    const double wide_cost = 2.0 * (double)pair_makespan(m_pairs, (int)cdiv64(N, WN), 1, npairs);
    const double pair_cost = 1.13 * (double)pair_makespan(m_pairs, (int)cdiv64(N, BN), 1, npairs);
    if (pair_cost < 0.95 * wide_cost) pl.kind = 1;
  }
  pl.n_tiles = (int)cdiv64(N, pl.kind == 2 ? WN : BN);
  if (splits_hint <= 0) {
    pl.tiles_per_split = 1;
  } else {
    pl.tiles_per_split = (int)cdiv64(pl.n_tiles, splits_hint);
    if (pl.kind == 0 && m_tiles == 1 && (is_tail(epi) || epi == EPI_DTAIL))
      pl.tiles_per_split = (int)cdiv64(pl.n_tiles, nsm);  // one CTA an SM, one round
    if ((is_dlogits(epi) || is_tail(epi)) && pl.kind != 0 && persistent && balance_splits_enabled())
      pl.tiles_per_split = balanced_tiles_per_split(m_tiles, pl.n_tiles, splits_hint, npairs);
  }
  pl.splits = (int)cdiv64(pl.n_tiles, pl.tiles_per_split);
  return pl;
}

// A chunk's dH may be split into at most kMaxDhSplitK K ranges, whose fp32 partials take at most
// kSplitKPartElems elements (512 MB) of the backward workspace.
constexpr int kMaxDhSplitK = 16;
constexpr int64_t kSplitKPartElems = 128ll << 20;

// K ranges for a chunk's dH = dS W.  Every 256 x 512 dH tile reduces over the whole vocabulary, so
// few row tiles leave few units: the 0.6B head's 10,066 active rows are 40 row pairs x 2 column
// tiles = 80 units for 74 pairs, two rounds where the mean is 1.08.  With ks K ranges there are
// ks times the units, each storing an fp32 partial; a second kernel sums the partials in a fixed
// order.  ks minimises the busiest pair's work plus the partials' HBM write and read (in units of
// one full-vocabulary 256 x 256 tile), and is taken when that beats the undivided choice of
// plan_k1 (256 x 512, or 256 x 256 pairs) by 5%.  1 = no split.
// many: weigh K ranges for launches of more than two rounds of units too (the row losses' rule; 5461 rows x
// 4096 are 176 units, 2.4 rounds of the pairs: two ranges took 2% off the whole step).
int dh_split_k(int64_t m_tiles, int H, int V, int64_t rows, int64_t part_elems, int nsm, bool many = false) {
  const int64_t forced = tuning(IKRL_TUNE_DH_SPLIT_K);
  if (forced == 0 || forced == 1) return 1;
  if (!use_pairs() || !use_wide(V) || !persistent_pairs()) return 1;
  const int64_t nk = cdiv64(V, BK);
  auto fits = [&](int64_t ks) { return ks * rows * H <= part_elems && nk / ks >= 32; };
  if (forced > 1) {
    int64_t ks = std::min<int64_t>(forced, kMaxDhSplitK);
    while (ks > 1 && !fits(ks)) --ks;
    return (int)ks;
  }
  const int64_t P = std::max(1, nsm / 2);
  const int64_t m_pairs = (m_tiles + 1) / 2;
  const int64_t U = m_pairs * cdiv64(H, WN);
  if (U >= (many ? 8 : 2) * P) return 1;
  const double tile_s = 2.0 * BN * BN * (double)V / (1.4e15 / (double)P);  // one tile on one pair
  const double elem_s = 8.0 / 6.0e12;                                       // fp32 written and read
  auto cost = [&](int64_t ks) {
    return 2.0 * (double)cdiv64(U * ks, P) / (double)ks + (double)(ks * rows * H) * elem_s / tile_s;
  };
  const double undivided = std::min(2.0 * (double)cdiv64(U, P),
                                    1.13 * (double)pair_makespan(m_pairs, (int)cdiv64(H, BN), 1, P));
  int64_t best_ks = 1;
  double best = undivided;
  for (int64_t ks = 2; ks <= kMaxDhSplitK && fits(ks); ++ks) {
    const double c = cost(ks);
    if (c < best) { best = c; best_ks = ks; }
  }
  return best < 0.95 * undivided ? (int)best_ks : 1;
}

// dH rows of a split dH: out = bf16(part[0] + part[1] + ... + part[ks-1]), summed in that order.
// n4: float4 groups of one partial (rows * H / 4); the partials are n4 groups apart.
__global__ void splitk_sum_kernel(const float4* __restrict__ part, int64_t n4, int ks, uint2* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n4; i += (int64_t)gridDim.x * blockDim.x) {
    float4 a = part[i];
#pragma unroll 8
    for (int s = 1; s < ks; ++s) {
      const float4 b = part[(int64_t)s * n4 + i];
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
    out[i] = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
  }
}

// Launch one K1 GEMM with the kernel plan_k1 selects, filling in the tile ranges; p.splits holds
// the count actually used.
// c_store: tensor map of the dS chunk for the wide kernel's TMA stores (DLOGITS), or null.
template <int EPI, bool A_MN, bool B_MN>
int launch_k1(const CUtensorMap& a_single, const CUtensorMap& b_single, const CUtensorMap& a_pair,
              const CUtensorMap& b_pair, GemmParams& p, int m_tiles, int splits_hint, cudaStream_t s,
              const CUtensorMap* c_store = nullptr) {
  int dev = 0, nsm = kNumSMs;
  IKRL_CUDA(cudaGetDevice(&dev));
  IKRL_CUDA(cudaDeviceGetAttribute(&nsm, cudaDevAttrMultiProcessorCount, dev));
  const K1Plan pl = plan_k1(EPI, m_tiles, p.N, p.K, splits_hint, nsm);
  const int kind = pl.kind;
  p.n_tiles = pl.n_tiles;
  p.tiles_per_split = pl.tiles_per_split;
  p.splits = pl.splits;
  p.split_major = 1;
  p.part_sets = p.splits * (kind == 2 ? kWideGroups : 1);
  if constexpr (is_tail(EPI))
    IKRL_REQUIRE(p.part_sets <= p.part_cap, IKRL_ERR_WORKSPACE, "%d partial sets, room for %d", p.part_sets, p.part_cap);
  {
    // L2 policy of the A and B loads of the wide kernel (0 normal, 1 evict-last, 2 evict-first),
    // IKRL_TUNE_L2_POLICY = 10 * a + b.  Default: A (re-read by every tile of a unit) evict-last,
    // B normal; evict-first on B measured 40% more DRAM traffic.
    const int64_t pol = tuning(IKRL_TUNE_L2_POLICY);
    p.a_policy = kind == 2 ? 1 : 0;
    p.b_policy = 0;
    if (pol >= 0) {
      p.a_policy = (int)(pol / 10);
      p.b_policy = (int)(pol % 10);
    }
  }
  if (kind == 2) return launch_gemm_pair<EPI, A_MN, B_MN, true>(a_pair, b_pair, c_store, p, m_tiles, s);
  if constexpr (EPI == EPI_STORE_TMA) return IKRL_ERR_UNSUPPORTED;  // plan_k1 gives it the wide kernel
  else if (kind == 1) return launch_gemm_pair<EPI, A_MN, B_MN, false>(a_pair, b_pair, nullptr, p, m_tiles, s);
  else return launch_gemm<EPI, A_MN, B_MN>(a_single, b_single, p, m_tiles, s);
}

int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Vocab splits for the row-sweeping GEMMs: enough that the row blocks resident at once keep their
// A tiles in L2 (about 24 MB of hidden rows), and enough CTAs to fill the GPU.
int choose_splits(int64_t m_tiles, int n_tiles, int H) {
  // L2 share for the A rows of the units in flight.  Long reductions (the wide kernel, whose A
  // loads are marked evict-last and whose pairs are paced) keep more rows resident and split the
  // vocabulary less: at H = 4096, 40 MB gives 4 splits.
  int64_t budget_mb = H >= 2048 ? 40 : 24;
  if (tuning(IKRL_TUNE_L2_BUDGET_MB) > 0) budget_mb = tuning(IKRL_TUNE_L2_BUDGET_MB);
  const int64_t resident_rows_budget = (budget_mb << 20) / (2ll * H);   // rows whose A tiles fit the budget
  const int64_t blocks_resident = std::max<int64_t>(1, resident_rows_budget / BM);
  int64_t s = cdiv64(kNumSMs, std::min<int64_t>(blocks_resident, m_tiles));
  s = std::max<int64_t>(s, cdiv64(2 * kNumSMs, m_tiles));
  s = std::min<int64_t>(s, n_tiles);
  return (int)std::max<int64_t>(1, s);
}

struct FwdLayout {
  size_t err_off, pm_off, ps_off, pt_off, total;
  int splits, tps;
};

FwdLayout fwd_layout(int64_t N, int H, int V) {
  FwdLayout L;
  const int64_t m_tiles = cdiv64(N, BM);
  const int n_tiles = (int)cdiv64(V, BN);
  int s = choose_splits(m_tiles, n_tiles, H);
  L.tps = (int)cdiv64(n_tiles, s);
  L.splits = (int)cdiv64(n_tiles, L.tps);
  auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
  L.err_off = 0;
  L.pm_off = 256;
  // up to kWideGroups partial sets per split (the wide kernel's column groups)
  L.ps_off = al(L.pm_off + (size_t)kWideGroups * L.splits * N * 4);
  L.pt_off = al(L.ps_off + (size_t)kWideGroups * L.splits * N * 4);
  L.total = al(L.pt_off + (size_t)N * 4);
  return L;
}

struct BwdLayout {
  size_t err_off, ds_off, dw_off, total;
  int64_t chunk, lds;
  bool need_dw32;
  // active-row compaction (rows whose upstream gradient is exactly zero are skipped)
  size_t cnt_off, nact_off, idx_off, pos_off, idc_off, lsec_off, gc_off, hc_off, part_off;
  int64_t part_elems;
  int cblocks;
};

constexpr int kCompactRows = 2048;    // rows per block of the compaction kernels
constexpr int kCompactThreads = 256;

BwdLayout bwd_layout(int64_t N, int H, int V, int64_t chunk_rows, int dweight_dtype, int accumulate) {
  BwdLayout L;
  int64_t c = chunk_rows > 0 ? chunk_rows : N;
  c = std::min<int64_t>(c, N);
  if (c < N) c = std::max<int64_t>(BM, (c / BM) * BM);
  L.chunk = std::max<int64_t>(c, 1);
  L.lds = cdiv64(V, 64) * 64;
  const int64_t nchunks = cdiv64(N, L.chunk);
  L.need_dw32 = (dweight_dtype == IKRL_DTYPE_BF16) && (nchunks > 1 || accumulate);
  auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
  L.err_off = 0;
  L.ds_off = 256;
  L.dw_off = al(L.ds_off + (size_t)L.chunk * L.lds * 2);
  size_t o = L.dw_off + (L.need_dw32 ? al((size_t)V * H * 4) : 0);
  L.cblocks = (int)std::max<int64_t>(1, cdiv64(N, kCompactRows));
  L.cnt_off = o;   o = al(o + (size_t)2 * L.cblocks * 4);
  L.nact_off = o;  o = al(o + 16);
  L.idx_off = o;   o = al(o + (size_t)N * 4);
  L.pos_off = o;   o = al(o + (size_t)N * 4);
  L.idc_off = o;   o = al(o + (size_t)N * 8);
  L.lsec_off = o;  o = al(o + (size_t)N * 4);
  L.gc_off = o;    o = al(o + (size_t)N * 4);
  L.hc_off = o;    o = al(o + (size_t)N * H * 2);
  // fp32 partials of a dH split into K ranges (few row tiles only; see dh_split_k)
  L.part_elems = std::min<int64_t>(kSplitKPartElems, (int64_t)kMaxDhSplitK * std::min<int64_t>(N, L.chunk) * H);
  L.part_off = o;  o = al(o + (size_t)L.part_elems * 4);
  L.total = o;
  return L;
}

// ---- active-row compaction -------------------------------------------------------------------
//
// A row contributes to dHidden and dW only through g * (onehot - softmax): rows whose upstream
// gradient g is exactly zero (tokens outside the response mask) and ignore_index rows contribute
// exact zeros.  The backward gathers the other rows, in row order, into a dense block, runs the
// three GEMMs on that block only, and scatters dHidden back (zero rows elsewhere).  NaN gradients
// count as active, so they propagate as in the dense computation.

__device__ __forceinline__ bool row_active(const float* __restrict__ g, const int64_t* __restrict__ ids, int64_t r) {
  return ids[r] != -100 && g[r] != 0.f;
}

// Rows are in two classes when the forward cached logits: active rows with a cache slot (their dS
// comes from the cache) and the other active rows (their dS is recomputed by the GEMM).  The
// compaction puts the cached class first, each class in row order.  Without a cache (slot null)
// every active row is in the second class.
__device__ __forceinline__ bool row_cached(const int* __restrict__ slot, int64_t r) {
  return slot != nullptr && slot[r] >= 0;
}

// counts[b] = cached active rows of block b, counts[nb + b] = the other active rows.
__global__ void __launch_bounds__(kCompactThreads) active_count_kernel(const float* __restrict__ g,
                                                                       const int64_t* __restrict__ ids,
                                                                       const int* __restrict__ slot, int64_t N,
                                                                       int* __restrict__ counts) {
  __shared__ int wsum[2][kCompactThreads / 32];
  const int64_t r0 = (int64_t)blockIdx.x * kCompactRows;
  int cc = 0, cu = 0;
  for (int i = threadIdx.x; i < kCompactRows; i += blockDim.x) {
    const int64_t r = r0 + i;
    if (r < N && row_active(g, ids, r)) {
      if (row_cached(slot, r)) ++cc;
      else ++cu;
    }
  }
  cc = warp_sum(cc);
  cu = warp_sum(cu);
  if ((threadIdx.x & 31) == 0) {
    wsum[0][threadIdx.x >> 5] = cc;
    wsum[1][threadIdx.x >> 5] = cu;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int tc = 0, tu = 0;
    for (int w = 0; w < kCompactThreads / 32; ++w) {
      tc += wsum[0][w];
      tu += wsum[1][w];
    }
    counts[blockIdx.x] = tc;
    counts[gridDim.x + blockIdx.x] = tu;
  }
}

// Block b writes its cached active rows after those of blocks 0..b-1, and its other active rows
// after all cached rows and the other rows of blocks 0..b-1, each in row order: idx[k] = row,
// pos[row] = k (-1 for skipped rows), and the compacted ids / lse / g.  The last block writes
// n_out[0] = active rows and n_out[1] = cached active rows.
__global__ void __launch_bounds__(kCompactThreads) compact_rows_kernel(
    const float* __restrict__ g, const int64_t* __restrict__ ids, const int* __restrict__ slot,
    const float* __restrict__ lse, int64_t N, const int* __restrict__ counts, int* __restrict__ idx,
    int* __restrict__ pos, int64_t* __restrict__ ids_c, float* __restrict__ lse_c, float* __restrict__ g_c,
    int64_t* __restrict__ n_out) {
  constexpr int kWarps = kCompactThreads / 32;
  __shared__ int wt[2][kWarps];
  __shared__ int s_base[3];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nb = (int)gridDim.x;
  int pc = 0, pu = 0, tc = 0;
  for (int b = threadIdx.x; b < nb; b += blockDim.x) {
    const int c = counts[b];
    tc += c;
    if (b < (int)blockIdx.x) {
      pc += c;
      pu += counts[nb + b];
    }
  }
  pc = warp_sum(pc);
  pu = warp_sum(pu);
  tc = warp_sum(tc);
  __shared__ int red[3][kWarps];
  if (lane == 0) {
    red[0][warp] = pc;
    red[1][warp] = pu;
    red[2][warp] = tc;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int a = 0, b2 = 0, c2 = 0;
    for (int w = 0; w < kWarps; ++w) {
      a += red[0][w];
      b2 += red[1][w];
      c2 += red[2][w];
    }
    s_base[0] = a;       // cached rows before this block
    s_base[1] = c2 + b2; // other rows: after every cached row and the earlier blocks' other rows
    s_base[2] = c2;      // cached rows in total
  }
  __syncthreads();
  int base_c = s_base[0], base_u = s_base[1];
  const int64_t r0 = (int64_t)blockIdx.x * kCompactRows;
  for (int off = 0; off < kCompactRows; off += kCompactThreads) {
    const int64_t r = r0 + off + threadIdx.x;
    const bool act = r < N && row_active(g, ids, r);
    const bool cached = act && row_cached(slot, r);
    const unsigned bc = __ballot_sync(0xffffffffu, cached);
    const unsigned bu = __ballot_sync(0xffffffffu, act && !cached);
    __syncthreads();  // wt is reused
    if (lane == 0) {
      wt[0][warp] = __popc(bc);
      wt[1][warp] = __popc(bu);
    }
    __syncthreads();
    int before_c = 0, before_u = 0, total_c = 0, total_u = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      before_c += (w < warp) ? wt[0][w] : 0;
      before_u += (w < warp) ? wt[1][w] : 0;
      total_c += wt[0][w];
      total_u += wt[1][w];
    }
    if (act) {
      const unsigned below = (1u << lane) - 1u;
      const int k = cached ? base_c + before_c + __popc(bc & below) : base_u + before_u + __popc(bu & below);
      idx[k] = (int)r;
      pos[r] = k;
      ids_c[k] = ids[r];
      lse_c[k] = lse[r];
      g_c[k] = g[r];
    } else if (r < N) {
      pos[r] = -1;
    }
    base_c += total_c;
    base_u += total_u;
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
    n_out[0] = base_u;  // the last block's other rows end at the total active count
    n_out[1] = s_base[2];
  }
}

// Cache slots of the forward: rows with cache_mask[r] != 0 (all rows when null) and a target,
// numbered in row order; rows past `cap` of them get -1.  counts[b] = such rows of block b.
__device__ __forceinline__ bool row_wants_cache(const uint8_t* __restrict__ mask, const int64_t* __restrict__ ids,
                                                int64_t r) {
  return ids[r] != -100 && (mask == nullptr || mask[r] != 0);
}

__global__ void __launch_bounds__(kCompactThreads) cache_count_kernel(const uint8_t* __restrict__ mask,
                                                                      const int64_t* __restrict__ ids, int64_t N,
                                                                      int* __restrict__ counts) {
  __shared__ int wsum[kCompactThreads / 32];
  const int64_t r0 = (int64_t)blockIdx.x * kCompactRows;
  int c = 0;
  for (int i = threadIdx.x; i < kCompactRows; i += blockDim.x) {
    const int64_t r = r0 + i;
    if (r < N && row_wants_cache(mask, ids, r)) ++c;
  }
  c = warp_sum(c);
  if ((threadIdx.x & 31) == 0) wsum[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    int t = 0;
    for (int w = 0; w < kCompactThreads / 32; ++w) t += wsum[w];
    counts[blockIdx.x] = t;
  }
}

__global__ void __launch_bounds__(kCompactThreads) cache_slot_kernel(const uint8_t* __restrict__ mask,
                                                                     const int64_t* __restrict__ ids, int64_t N,
                                                                     const int* __restrict__ counts, int64_t cap,
                                                                     int* __restrict__ slot) {
  constexpr int kWarps = kCompactThreads / 32;
  __shared__ int wtot[kWarps];
  __shared__ int s_base;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int part = 0;
  for (int b = threadIdx.x; b < (int)blockIdx.x; b += blockDim.x) part += counts[b];
  part = warp_sum(part);
  if (lane == 0) wtot[warp] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    int t = 0;
    for (int w = 0; w < kWarps; ++w) t += wtot[w];
    s_base = t;
  }
  __syncthreads();
  int base = s_base;
  const int64_t r0 = (int64_t)blockIdx.x * kCompactRows;
  for (int off = 0; off < kCompactRows; off += kCompactThreads) {
    const int64_t r = r0 + off + threadIdx.x;
    const bool want = r < N && row_wants_cache(mask, ids, r);
    const unsigned bal = __ballot_sync(0xffffffffu, want);
    __syncthreads();
    if (lane == 0) wtot[warp] = __popc(bal);
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      before += (w < warp) ? wtot[w] : 0;
      total += wtot[w];
    }
    if (r < N) {
      const int k = base + before + __popc(bal & ((1u << lane) - 1u));
      slot[r] = (want && k < cap) ? k : -1;
    }
    base += total;
  }
}

// dS of cached rows: for chunk row k (compacted row c0 + k, original row idx[c0 + k]) and column
// j < V, dS = g * ([j == t] - q * 2^(m - lse log2e)), with q the cached bf16 numerator and m its
// chunk maximum.  Block row y handles chunk rows y, y + gridDim.y, ...; a thread takes
// kDsUnroll groups of eight columns, 256 groups apart, and issues their 16-byte loads before any
// store; V must be a multiple of 8.
constexpr int kDsUnroll = 4;
__global__ void __launch_bounds__(256) ds_from_cache_kernel(
    const uint16_t* __restrict__ cache_q, const float* __restrict__ cache_m, int64_t ld_cache, int n_mchunks,
    const int* __restrict__ slot, const int* __restrict__ idx, const int64_t* __restrict__ ids_c,
    const float* __restrict__ lse_c, const float* __restrict__ g_c, int64_t c0, int64_t rows, int V,
    int64_t id_offset, uint16_t* __restrict__ ds, int64_t ld_ds) {
  const int vec = V >> 3;
  for (int64_t k = blockIdx.y; k < rows; k += gridDim.y) {
    const int64_t kc = c0 + k;
    const int64_t sl = slot[idx[kc]];
    const float lse2 = lse_c[kc] * kLog2e;
    const float gv = g_c[kc];
    const int64_t t = ids_c[kc] - id_offset;
    const uint16_t* qrow = cache_q + sl * ld_cache;
    const float* mrow = cache_m + sl * n_mchunks;
    uint16_t* drow = ds + k * ld_ds;
    for (int jb = blockIdx.x * blockDim.x * kDsUnroll + threadIdx.x; jb < vec;
         jb += gridDim.x * blockDim.x * kDsUnroll) {
      uint4 qv[kDsUnroll];
      float mv[kDsUnroll];
#pragma unroll
      for (int u = 0; u < kDsUnroll; ++u) {
        const int jv = jb + u * (int)blockDim.x;
        if (jv < vec) {
          qv[u] = *reinterpret_cast<const uint4*>(qrow + (jv << 3));
          mv[u] = mrow[jv >> 2];
        }
      }
#pragma unroll
      for (int u = 0; u < kDsUnroll; ++u) {
        const int jv = jb + u * (int)blockDim.x;
        if (jv >= vec) break;
        const int j0 = jv << 3;
        const float sc = fast_exp2(mv[u] - lse2);
        const uint32_t w[4] = {qv[u].x, qv[u].y, qv[u].z, qv[u].w};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = bf16lo(w[e]) * sc, p1 = bf16hi(w[e]) * sc;
          const float d0 = gv * (((int64_t)(j0 + 2 * e) == t ? 1.f : 0.f) - p0);
          const float d1 = gv * (((int64_t)(j0 + 2 * e + 1) == t ? 1.f : 0.f) - p1);
          o[e] = pack_bf16x2(d0, d1);
        }
        *reinterpret_cast<uint4*>(drow + j0) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
}

// The same for a row loss: dS = g (coef q 2^(c (m - ref)) + level), then g grad at the row's entries,
// written behind a barrier by the block that holds their columns.  slot null: row r has slot r; idx null:
// chunk row k is row c0 + k.  Rows without a gradient (or a slot) are zeros.  TWO: dS in two bf16 terms, what the
// rounding of the first leaves (rounded itself) `rows` rows below; otherwise dS times mul[c0 + k] in fp16.
template <bool TWO>
__global__ void __launch_bounds__(256) dtail_from_cache_kernel(
    const uint16_t* __restrict__ cache_q, const float* __restrict__ cache_m, int64_t ld_cache, int n_mchunks,
    const int* __restrict__ slot, const int* __restrict__ idx, const float* __restrict__ dloss,
    const int64_t* __restrict__ row_ids, const float* __restrict__ refs, const float* __restrict__ coefs,
    const int* __restrict__ cols, const float* __restrict__ grads, const float* __restrict__ mul, int K, float level,
    float c, int64_t c0, int64_t rows, int V, uint16_t* __restrict__ ds, int64_t ld_ds) {
  const int vec = V >> 3;
  const int jb = blockIdx.x * blockDim.x * kDsUnroll + threadIdx.x;  // gridDim.x covers the columns
  for (int64_t k = blockIdx.y; k < rows; k += gridDim.y) {
    const int64_t r = idx ? idx[c0 + k] : c0 + k;
    const int64_t sl = slot ? slot[r] : r;
    float g = dloss[r];
    const float ref = refs[r], coef = coefs[r];
    const bool on = sl >= 0 && g != 0.f && row_ids[r] != kRowNone;
    if constexpr (!TWO) g *= mul[c0 + k];
    const float gs = g * coef, lv = on ? g * level : 0.f;
    const uint16_t* qrow = cache_q + (on ? sl : 0) * ld_cache;
    const float* mrow = cache_m + (on ? sl : 0) * n_mchunks;
    uint16_t* drow = ds + k * ld_ds;
    uint16_t* lrow = ds + (rows + k) * ld_ds;
    uint4 qv[kDsUnroll];
    float mv[kDsUnroll];
#pragma unroll
    for (int u = 0; u < kDsUnroll; ++u) {
      const int jv = jb + u * (int)blockDim.x;
      qv[u] = make_uint4(0u, 0u, 0u, 0u);
      mv[u] = 0.f;
      if (on && jv < vec) {
        qv[u] = *reinterpret_cast<const uint4*>(qrow + (jv << 3));
        mv[u] = mrow[jv >> 2];
      }
    }
#pragma unroll
    for (int u = 0; u < kDsUnroll; ++u) {
      const int jv = jb + u * (int)blockDim.x;
      if (jv >= vec) break;
      const float sc = on ? gs * fast_exp2((mv[u] - ref) * c) : 0.f;
      const uint32_t w[4] = {qv[u].x, qv[u].y, qv[u].z, qv[u].w};
      uint32_t o[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
        const float d0 = fmaf(q.x, sc, lv), d1 = fmaf(q.y, sc, lv);
        if constexpr (TWO) {
          o[e] = pack_bf16x2(d0, d1);
          lo[e] = pack_bf16x2(d0 - bf16lo(o[e]), d1 - bf16hi(o[e]));
        } else {
          o[e] = pack_f16x2(d0, d1);
        }
      }
      *reinterpret_cast<uint4*>(drow + (jv << 3)) = make_uint4(o[0], o[1], o[2], o[3]);
      if constexpr (TWO) *reinterpret_cast<uint4*>(lrow + (jv << 3)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    __syncthreads();
    if (on) {
      const int lo = (int)(blockIdx.x * blockDim.x * kDsUnroll) << 3, hi = lo + ((int)blockDim.x * kDsUnroll << 3);
      for (int e = threadIdx.x; e < K; e += blockDim.x) {
        const int col = cols[r * K + e];
        if (col == kNoEntry || col < lo || col >= hi) continue;
        const float d = g * grads[r * K + e];
        if constexpr (TWO) {
          drow[col] = f32_to_bf16_rn(d);
          lrow[col] = f32_to_bf16_rn(d - bf16_to_f32(drow[col]));
        } else {
          drow[col] = __half_as_ushort(__float2half_rn(d));
        }
      }
    }
  }
}

// Column ranges of a GEMM over gathered rows: n_tiles column tiles, `tiles_per_split` and `splits` as planned
// for all rows.  least > 0: from `least` to `most` ranges for the rows there are, on npairs CTA pairs.
struct LiveSplit {
  int n_tiles, tiles_per_split, splits, least, most, npairs, groups;
};

// From the numbers pos[r] that cache_slot_kernel gave the rows of a row loss that are not kRowNone:
// idx[pos[r]] = r, slot[r] = pos[r] where that is below the cache's slots (slot may be null), and the plan.
// The ranges are dealt to the pairs in rounds; fewest tiles on the busiest pair wins, a further range
// (the weights are then read more often) being worth 1%.  Of 16384 rows of 1024 against 151936 columns 10923
// count: 3.28 ms in the ranges planned for all rows, 3.05 ms in these.
__global__ void row_index_kernel(const int* __restrict__ pos, int64_t N, int64_t cap, int* __restrict__ idx,
                                 int* __restrict__ slot, const int* __restrict__ counts, int n_counts, LiveSplit ls,
                                 int* __restrict__ plan) {
  const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (blockIdx.x == 0 && threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int n = 0;
    for (int b = lane; b < n_counts; b += 32) n += counts[b];
    n = __reduce_add_sync(0xffffffffu, n);
    int tps = ls.tiles_per_split, splits = ls.splits;
    if (ls.least > 0) {
      const unsigned m_pairs = (unsigned)(n + 2 * BM - 1) / (2 * BM);
      unsigned best = 0xffffffffu, best_sp = 0xffffffffu;
      for (int sp = ls.least + lane; sp <= ls.most; sp += 32) {
        const unsigned t = (ls.n_tiles + sp - 1) / sp, rounds = (m_pairs * sp + ls.npairs - 1) / ls.npairs;
        const unsigned cost = rounds * t * (100 + sp);
        if (cost < best) {
          best = cost;
          best_sp = sp;
        }
      }
      const unsigned all = __reduce_min_sync(0xffffffffu, best);
      const int sp = (int)__reduce_min_sync(0xffffffffu, best == all ? best_sp : 0xffffffffu);
      tps = (ls.n_tiles + sp - 1) / sp;
      splits = (ls.n_tiles + tps - 1) / tps;
    }
    if (lane == 0) {
      plan[LIVE_ROWS] = n;
      plan[LIVE_TILES_PER_SPLIT] = tps;
      plan[LIVE_SPLITS] = splits;
      plan[LIVE_SETS] = splits * ls.groups;
    }
  }
  if (r >= N) return;
  const int k = pos[r];
  if (k >= 0) idx[k] = (int)r;
  if (slot != nullptr) slot[r] = k < cap ? k : -1;
}

// h_c[k] = h[idx[k]] for k < *n.
__global__ void gather_live_rows_kernel(const uint4* __restrict__ h, const int* __restrict__ idx,
                                        const int* __restrict__ n, int vec_per_row, uint4* __restrict__ h_c) {
  const int64_t total = (int64_t)*n * vec_per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t k = i / vec_per_row;
    const int c = (int)(i - k * vec_per_row);
    h_c[i] = h[(int64_t)idx[k] * vec_per_row + c];
  }
}

// h . w by one warp, in every lane: 32-bit sums of exact products.
__device__ __forceinline__ float warp_dot(const uint4* __restrict__ a, const uint4* __restrict__ b, int vec_per_row) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
  for (int v = threadIdx.x & 31; v < vec_per_row; v += 32) {
    const uint4 x = a[v], y = b[v];
    s0 = fmaf(bf16lo(x.x), bf16lo(y.x), s0);
    s1 = fmaf(bf16hi(x.x), bf16hi(y.x), s1);
    s0 = fmaf(bf16lo(x.y), bf16lo(y.y), s0);
    s1 = fmaf(bf16hi(x.y), bf16hi(y.y), s1);
    s0 = fmaf(bf16lo(x.z), bf16lo(y.z), s0);
    s1 = fmaf(bf16hi(x.z), bf16hi(y.z), s1);
    s0 = fmaf(bf16lo(x.w), bf16lo(y.w), s0);
    s1 = fmaf(bf16hi(x.w), bf16hi(y.w), s1);
  }
  return warp_sum(s0 + s1);
}

// The logits at the entries, xk[r][e] = h_r . w_col, one warp an entry.  The GEMM's accumulators cut every
// partial sum to 24 bits towards zero, which takes about 1e-9 H of a logit away; a distilled student's likely
// tokens are mostly among the entries, so this leaves little of it (loss of an 8B-sized head against 64 bits:
// 1.3e-5 -> 2.5e-6).  A cross entropy takes its target's logit from here where exact_tops_kernel deals with its
// tail as well, and from the accumulators below kExactTopsHidden: target and tail are then short by about the
// same.
__global__ void __launch_bounds__(256) entry_logits_kernel(const uint4* __restrict__ h, const uint4* __restrict__ w,
                                                           const int* __restrict__ cols, int64_t n, int K,
                                                           int vec_per_row, float* __restrict__ xk) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= n) return;
  const int col = cols[i];
  if (col == kNoEntry) return;
  const float s = warp_dot(h + i / K * vec_per_row, w + (int64_t)col * vec_per_row, vec_per_row);
  if ((threadIdx.x & 31) == 0) xk[i] = s;
}

// The tail's likely tokens, with logits as exact as the entries': of each partial set whose largest column holds
// 2^-10 of its row's sum or more, that column's share is taken from warp_dot instead of the accumulators.  WARPS warps
// a row, as row_losses_kernel; they share the columns found.  The other columns are many and unlikely, and their
// logits small, so what the accumulators cut of them does not show (a set's second likely token keeps its cut logit:
// 14 rows of 1992 against 1174 columns, five sets, stay at 2e-6).  Cross entropy against 64 bits: 4 rows of 3904
// against 17394 columns 3e-6 -> 5e-7, 16384 of 1024 against 151936 1.2e-6 -> 2e-7 (38 us for 8192 of those).
constexpr int kExactTopsHidden = 1024;
constexpr float kTopShare = 1.f / 1024.f;
template <int WARPS>
__global__ void __launch_bounds__(128) exact_tops_kernel(const uint4* __restrict__ h, const uint4* __restrict__ w,
                                                         int vec_per_row, const float* __restrict__ part_m,
                                                         const int* __restrict__ part_c, float* __restrict__ part_s,
                                                         int sets, const int* __restrict__ sets_dev,
                                                         const int* __restrict__ pos,
                                                         const int64_t* __restrict__ row_ids,
                                                         const float* __restrict__ xk, const int* __restrict__ cols,
                                                         int K, int64_t N, int V, float c,
                                                         const int* __restrict__ err) {
  static_assert(WARPS == 1 || WARPS == 4, "a block's four warps take four rows or one");
  constexpr int kList = 256;  // sets taken at a time
  __shared__ float s_m[4], s_s[4];
  __shared__ int s_list[4 / WARPS][kList], s_count[4 / WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (4 / WARPS) + (WARPS == 1 ? warp : 0);
  if (r >= N || row_ids[r] != kRowLive || *err != 0) return;  // after an error the sets may hold anything
  const int64_t at = pos ? pos[r] : r;
  if (sets_dev != nullptr) sets = *sets_dev;
  const int first = WARPS == 1 ? lane : (int)threadIdx.x;
  int* list = s_list[WARPS == 1 ? warp : 0];
  int& count = s_count[WARPS == 1 ? warp : 0];
  auto sync = [&]() {
    if constexpr (WARPS == 1) __syncwarp();
    else __syncthreads();
  };
  // the row's maximum m and its sum s of 2^(c (x - m)), over sets and entries
  float m = -INFINITY, s = 0.f;
  auto merge = [&](float m2, float s2) {
    const float mm = fmaxf(m, m2);
    if (mm > -INFINITY) {
      s = s * exp2f((m - mm) * c) + s2 * exp2f((m2 - mm) * c);
      m = mm;
    }
  };
#pragma unroll 4
  for (int q = first; q < sets; q += 32 * WARPS)
    merge(part_m[(int64_t)q * N + at], part_s[(int64_t)q * N + at]);
  for (int k = first; k < K; k += 32 * WARPS)
    if (cols[r * K + k] != kNoEntry) merge(xk[r * K + k], 1.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    merge(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if constexpr (WARPS == 4) {
    if (lane == 0) {
      s_m[warp] = m;
      s_s[warp] = s;
    }
    __syncthreads();
    m = -INFINITY;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) merge(s_m[i], s_s[i]);
  }
  const float least = s * kTopShare;
  const uint4* row = h + r * vec_per_row;
  for (int q0 = 0; q0 < sets; q0 += kList) {
    if (first == 0) count = 0;
    sync();
    for (int q = q0 + first; q < min(sets, q0 + kList); q += 32 * WARPS)
      if (exp2f((part_m[(int64_t)q * N + at] - m) * c) >= least) list[atomicAdd(&count, 1)] = q;  // not for NaN
    sync();
    for (int i = WARPS == 1 ? 0 : warp; i < count; i += WARPS) {
      const int64_t o = (int64_t)list[i] * N + at;
      const int col = part_c[o];
      if (col < 0 || col >= V) continue;
      const float x = warp_dot(row, w + (int64_t)col * vec_per_row, vec_per_row);
      if (lane == 0) part_s[o] += exp2f((x - part_m[o]) * c) - 1.f;
    }
    sync();
  }
}

// h_c[k] = h[idx[k]] for k < n, 16 bytes per thread.
__global__ void gather_rows_kernel(const uint4* __restrict__ h, const int* __restrict__ idx, int64_t n, int vec_per_row,
                                   uint4* __restrict__ h_c) {
  const int64_t total = n * vec_per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t k = i / vec_per_row;
    const int c = (int)(i - k * vec_per_row);
    h_c[i] = h[(int64_t)idx[k] * vec_per_row + c];
  }
}

// out[r] = pos[r] >= 0 ? src[pos[r]] : 0 for every row r < N, 16 bytes per thread.
__global__ void scatter_rows_kernel(const uint4* __restrict__ src, const int* __restrict__ pos, int64_t N,
                                    int vec_per_row, uint4* __restrict__ out) {
  const int64_t total = N * vec_per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / vec_per_row;
    const int c = (int)(i - r * vec_per_row);
    const int k = pos[r];
    out[i] = k >= 0 ? src[(int64_t)k * vec_per_row + c] : make_uint4(0u, 0u, 0u, 0u);
  }
}

// The backward of a row loss multiplies fp16 operands.  Rounded to bf16, dS took dH and dW to 1.4 times the error of
// their own final rounding (1.7 times where the upstream gradients are all alike and round the same way); in fp16 it
// leaves them at 1.0 times.  bf16 hidden rows and weights fit fp16 as they are, 8 bits in 11, and what fp16 lacks in
// range powers of two supply, which the epilogues take out again:
//   dS'_k = dS_k 2^(14 - e_k)        2^e_k above the largest |dS_k|
//   h'_k  = h_k 2^(e_k - 14 - X)     X one for all, so that the largest is below 2^15
//   W'    = W 2^(15 - e_W)           2^e_W above the largest |W|
//   dW    = 2^X dS'^T h',            dH_k = 2^(e_k + e_W - 29) dS'_k W'
// What lies more than 2^29 below its largest loses bits, one for each further 2, which is 2^-40 of that largest at most.
// Rows without a gradient are zeros in both operands (padding may hold NaN).  Infinities and NaN do not count for the
// ranges and stay what they are.  One more pass over W and a copy: 0.6 ms of 21 (8192 x 4096 x 151936).
struct RowRange {
  int* e;           // [rows] e_k, or kNoRange: no gradient
  float* mul;       // [rows] 2^(14 - e_k)
  float* gs;        // [rows] g coef mul and
  float* level;     // [rows] g level mul: what the dS epilogue multiplies and adds
  float* dh_scale;  // [rows] 2^(e_k + e_W - 29)
  unsigned* top;    // [0] largest e_k plus exponent of |h_k|, biased, 0: no row; [1] largest |W|, its bits;
  float* dw_scale;  // [1] 2^X
  uint16_t* h;      // [rows][H] h'
  uint16_t* w;      // [V][H] W'
};
constexpr int kNoRange = INT_MIN;
constexpr int kRangeBias = 1024;

// Exponent e with |x| < 2^e of a bf16 magnitude's bits (2^(e - 1) <= |x| too where x is a normal number).
__device__ __forceinline__ int bf16_exponent(uint32_t bits) { return (int)(bits >> 7) - 126; }
// e_W from the bits of the largest |W| (0: W is not wanted, or all of it is 0).
__device__ __forceinline__ int weight_exponent(unsigned bits) { return bits == 0 ? 0 : max(bf16_exponent(bits), -111); }
__device__ __forceinline__ uint32_t largest_finite(uint32_t m, uint32_t w) {
  const uint32_t lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
  m = max(m, lo < 0x7f80u ? lo : 0u);
  return max(m, hi < 0x7f80u ? hi : 0u);
}
__device__ __forceinline__ uint32_t largest_finite(uint32_t m, uint4 v) {
  return largest_finite(largest_finite(largest_finite(largest_finite(m, v.x), v.y), v.z), v.w);
}

// Ranges of rows [0, n): one warp a row (row idx[k], k itself when idx is null).
__global__ void __launch_bounds__(256) row_range_kernel(const float* __restrict__ dloss,
                                                        const int64_t* __restrict__ row_ids,
                                                        const float* __restrict__ coefs, const int* __restrict__ cols,
                                                        const float* __restrict__ grads, int K,
                                                        const int* __restrict__ idx, int64_t n, float level,
                                                        const uint4* __restrict__ h, int vec_per_row, RowRange R) {
  const int64_t k = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (k >= n) return;
  const int64_t r = idx ? idx[k] : k;
  const float g = dloss[r], coef = coefs[r];
  const bool on = g != 0.f && row_ids[r] != kRowNone;
  float most = fabsf(coef);
  for (int e = lane; e < K; e += 32)
    if (cols[r * K + e] != kNoEntry) most = fmaxf(most, fabsf(grads[r * K + e]));
  most = (warp_max(most) + fabsf(level)) * fabsf(g);
  uint32_t hm = 0;
  for (int i = lane; i < vec_per_row; i += 32) hm = largest_finite(hm, h[k * vec_per_row + i]);
  hm = __reduce_max_sync(0xffffffffu, hm);
  if (lane != 0) return;
  int e = kNoRange;
  float mul = 0.f;
  if (on) {
    e = 0;  // of an infinite or NaN gradient
    if (most < INFINITY) frexpf(most, &e);
    e = max(e, max(-100, -120 - weight_exponent(R.top[1])));  // 2^(e + e_W - 29) is a number
    mul = ldexpf(1.f, 14 - e);
    if (hm > 0) atomicMax(&R.top[0], (unsigned)(kRangeBias + e + bf16_exponent(hm)));
  }
  R.e[k] = e;
  R.mul[k] = mul;
  R.gs[k] = on ? g * mul * coef : 0.f;
  R.level[k] = on ? g * mul * level : 0.f;
}

__global__ void __launch_bounds__(256) weight_range_kernel(const uint4* __restrict__ w, int64_t n,
                                                           unsigned* __restrict__ top) {
  uint32_t m = 0;
#pragma unroll 4
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    m = largest_finite(m, w[i]);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0 && m > 0) atomicMax(top, m);
}

__device__ __forceinline__ uint32_t scale_to_f16(uint32_t w, float f) { return pack_f16x2(bf16lo(w) * f, bf16hi(w) * f); }
__device__ __forceinline__ uint4 scale_to_f16(uint4 v, float f) {
  return make_uint4(scale_to_f16(v.x, f), scale_to_f16(v.y, f), scale_to_f16(v.z, f), scale_to_f16(v.w, f));
}

// h' and the products' scales (h null: the scales only).
__global__ void __launch_bounds__(256) scale_rows_kernel(const uint4* __restrict__ h, int64_t n, int vec_per_row,
                                                         RowRange R) {
  // 2^X is a normal number: rows so small that it is not keep fewer bits of theirs
  const int X = min(max((int)R.top[0] - kRangeBias - 29, -126), 127);
  const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (first == 0) R.dw_scale[0] = ldexpf(1.f, X);
  const int ew = weight_exponent(R.top[1]);
  const int64_t total = h != nullptr ? n * vec_per_row : n;
  const int per = h != nullptr ? vec_per_row : 1;
  for (int64_t i = first; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t k = i / per;
    const int e = R.e[k];
    if (i == k * per) R.dh_scale[k] = e == kNoRange ? 1.f : ldexpf(1.f, e + ew - 29);
    if (h != nullptr)
      reinterpret_cast<uint4*>(R.h)[i] =
          e == kNoRange ? make_uint4(0u, 0u, 0u, 0u) : scale_to_f16(h[i], ldexpf(1.f, min(e - 14 - X, 126)));
  }
}

__global__ void __launch_bounds__(256) scale_weight_kernel(const uint4* __restrict__ w, int64_t n, RowRange R) {
  const float f = ldexpf(1.f, 15 - weight_exponent(R.top[1]));
#pragma unroll 4
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    reinterpret_cast<uint4*>(R.w)[i] = scale_to_f16(w[i], f);
}

// Row losses, backward: the gradient at the entries of chunk rows [c0, c0 + rows) goes over what the
// dS epilogue wrote there.  One block of threads per 256 entries.  TWO: two bf16 terms, the second `rows` rows
// below the first; otherwise times mul[c0 + k] in fp16.
template <bool TWO>
__global__ void ds_entries_kernel(const float* __restrict__ dloss, const int* __restrict__ cols,
                                  const float* __restrict__ grad, const float* __restrict__ mul, int K,
                                  const int* __restrict__ idx, int64_t c0, int64_t rows, uint16_t* __restrict__ ds,
                                  int64_t ld_ds) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= rows * K) return;
  const int64_t k = i / K;
  const int e = (int)(i - k * K);
  const int64_t r = idx ? idx[c0 + k] : c0 + k;
  const int col = cols[r * K + e];
  if (col == kNoEntry) return;
  const float g = dloss[r];
  if constexpr (TWO) {
    const float d = g != 0.f ? g * grad[r * K + e] : 0.f;
    const uint16_t hi = f32_to_bf16_rn(d);
    ds[k * ld_ds + col] = hi;
    ds[(rows + k) * ld_ds + col] = f32_to_bf16_rn(d - bf16_to_f32(hi));
  } else {
    ds[k * ld_ds + col] = __half_as_ushort(__float2half_rn(g != 0.f ? g * mul[c0 + k] * grad[r * K + e] : 0.f));
  }
}

// First launch of the backward of few rows, a block a row: clears the error word; with h2 the hidden rows
// twice, one under the other (the dW operand beside a dS of two terms); with gs what the dS epilogue multiplies and
// adds.  Rows without a gradient go in as zeros: padding may hold NaN, and 0 NaN would reach all of dW.
__global__ void __launch_bounds__(128) few_rows_kernel(const uint4* __restrict__ h, int vec_per_row, uint4* __restrict__ h2,
                                                       const float* __restrict__ dloss,
                                                       const int64_t* __restrict__ row_ids,
                                                       const float* __restrict__ coef, float level,
                                                       float* __restrict__ gs, float* __restrict__ level_out,
                                                       int* __restrict__ err) {
  const int64_t r = blockIdx.x;
  if (r == 0 && threadIdx.x == 0) *err = 0;
  const float g = dloss[r];
  const bool on = g != 0.f && row_ids[r] != kRowNone;
  if (gs != nullptr && threadIdx.x == 0) {
    gs[r] = on ? g * coef[r] : 0.f;
    level_out[r] = on ? g * level : 0.f;
  }
  if (h2 == nullptr) return;
  const uint4* from = h + r * vec_per_row;
  uint4* to = h2 + r * vec_per_row;
  uint4* below = to + (int64_t)gridDim.x * vec_per_row;
  for (int i = threadIdx.x; i < vec_per_row; i += blockDim.x)
    to[i] = below[i] = on ? from[i] : make_uint4(0u, 0u, 0u, 0u);
}

// dH of a dS of two terms: out = bf16(sum over K ranges of the partials of row r and of row rows + r).
// n4: float4 groups of the rows of one term, sets = 2 ks of them.  The sets are few groups long, so a group's
// sum is four threads' work, a quarter of the sets each, joined in a fixed order: at 74 sets of 96 x 1024 one
// thread's chain of loads took 19 us.
constexpr int kTermSumGroups = 64;
__global__ void __launch_bounds__(4 * kTermSumGroups) two_term_sum_kernel(const float4* __restrict__ part, int64_t n4,
                                                                          int sets, uint2* __restrict__ out) {
  __shared__ float4 sums[3][kTermSumGroups];
  const int t = threadIdx.x % kTermSumGroups, quarter = threadIdx.x / kTermSumGroups;
  const int64_t i = (int64_t)blockIdx.x * kTermSumGroups + t;
  const int s0 = sets * quarter / 4, s1 = sets * (quarter + 1) / 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < n4) {
#pragma unroll 8
    for (int s = s0; s < s1; ++s) {
      const float4 b = part[(int64_t)s * n4 + i];
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
  }
  if (quarter > 0) sums[quarter - 1][t] = a;
  __syncthreads();
  if (quarter > 0 || i >= n4) return;
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const float4 b = sums[q][t];
    a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
  }
  out[i] = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
}

// Row skipping is on unless IKRL_TUNE_SKIP_ZERO_ROWS = 0.
bool skip_zero_rows_enabled() { return tuning(IKRL_TUNE_SKIP_ZERO_ROWS) != 0; }

int check_common(const void* hidden, const void* weight, const int64_t* ids, int64_t N, int H, int V,
                 const char* what) {
  IKRL_REQUIRE(N >= 0 && H > 0 && V > 0, IKRL_ERR_INVALID_ARGUMENT, "%s: bad sizes N=%lld H=%d V=%d", what,
               (long long)N, H, V);
  IKRL_REQUIRE(H % 8 == 0, IKRL_ERR_ALIGNMENT, "%s: hidden size H=%d must be a multiple of 8 (16-byte rows)", what, H);
  IKRL_REQUIRE(N == 0 || (hidden && weight && ids), IKRL_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  IKRL_REQUIRE(N <= (int64_t)65535 * BM, IKRL_ERR_UNSUPPORTED, "%s: N=%lld rows exceeds one launch; chunk the call",
               what, (long long)N);
  return IKRL_OK;
}

}  // namespace
}  // namespace ikrl

using namespace ikrl;

// With no rows no kernel runs; the status word at the start of the workspace is still cleared so
// that ikrl_lmhead_status reads 0 after the call.
static int clear_status_word(void* ws, size_t ws_bytes, void* stream) {
  if (ws != nullptr && ws_bytes >= sizeof(int)) IKRL_CUDA(cudaMemsetAsync(ws, 0, sizeof(int), as_stream(stream)));
  return IKRL_OK;
}

// Logit cache of a forward (all null / 0: none).  mask: rows that may be cached (null = every row
// with a target); cap: cache slots; slot: [N] output, each row's slot or -1; q / m: the cache.
struct CacheArgs {
  const uint8_t* mask = nullptr;
  int64_t cap = 0;
  int* slot = nullptr;
  uint16_t* q = nullptr;
  float* m = nullptr;
};

// Workspace of the caching forward: the forward's, then the per-block counts of the slot numbering.
size_t cache_fwd_workspace_bytes(int64_t N, int H, int V) {
  const size_t base = fwd_layout(N, H, V).total;
  return base + ((((size_t)std::max<int64_t>(1, cdiv64(N, kCompactRows)) * 4) + 255) & ~size_t(255));
}

// A row loss of few rows runs its GEMMs on all of them, whichever count: up to 256, where one row pair of
// tiles costs the same however many of its rows count, and up to 1024 while the products are small enough
// that the compaction's host synchronisation and launches cost more than they save.  Its backward is
// lmhead_row_loss_bwd_few.  (Distillation forward and backward, a third without gradient: 300 rows of 512 against
// 32003 columns 176 us, 206 with the compaction; 512 of 1024 against 32000 229 / 259 us, without a cache 268 / 260.)
constexpr int64_t kRowLossDense = 256, kRowLossDenseMost = 1024;
constexpr double kRowLossDenseWork = 17179869184.0;  // N H V
static bool row_loss_dense(int64_t N, int H, int V) {
  return N <= kRowLossDense || (N <= kRowLossDenseMost && (double)N * H * V <= kRowLossDenseWork);
}

// Workspace of a row loss.  Its forward's: the GEMM's partial maxima, their columns, sums and sums of all logits
// (`sets` of each: the wide kernel's column groups of up to kBalanceMost times the forward's splits, which the balance
// rule may take), and the numbering of the rows that count with their hidden rows gathered.
static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
struct RowLossFwdLayout {
  size_t pm_off, ps_off, px_off, pc_off, counts_off, count_off, pos_off, idx_off, hc_off, total;
  int splits, sets;
  bool gather;  // the rows that count are gathered before the GEMM
};
static RowLossFwdLayout row_loss_fwd_layout(int64_t N, int H, int V) {
  RowLossFwdLayout L;
  L.splits = fwd_layout(N, H, V).splits;
  L.gather = !row_loss_dense(N, H, V);
  L.sets = kWideGroups * kBalanceMost * L.splits;
  const size_t part = align256((size_t)L.sets * N * 4);
  size_t o = 256;  // the error word
  L.pm_off = o; o += part;
  L.ps_off = o; o += part;
  L.px_off = o; o += part;
  L.pc_off = o; o += part;
  L.counts_off = o; o += align256((size_t)std::max<int64_t>(1, cdiv64(N, kCompactRows)) * 4);
  L.count_off = o; o += 256;
  L.pos_off = o; o += align256((size_t)N * 4);
  L.idx_off = o; o += align256((size_t)N * 4);
  L.hc_off = o; o += L.gather ? align256((size_t)N * H * 2) : 0;
  L.total = o;
  return L;
}

static int lmhead_fwd_impl(const char* what, const void* hidden, const void* weight, const int64_t* ids, int64_t N, int32_t H,
                    int32_t V, int64_t vocab_start, bool shard, float* logp, float* lse, void* ws, size_t ws_bytes,
                    void* stream, const CacheArgs& cache = CacheArgs()) {
  int rc = check_common(hidden, weight, ids, N, H, V, what);
  if (rc) return rc;
  if (N == 0) return clear_status_word(ws, ws_bytes, stream);
  IKRL_REQUIRE(logp != nullptr, IKRL_ERR_INVALID_ARGUMENT, "%s: output is NULL", what);
  const FwdLayout L = fwd_layout(N, H, V);
  IKRL_REQUIRE(ws != nullptr && ws_bytes >= L.total, IKRL_ERR_WORKSPACE,
               "%s: workspace %zu < %zu bytes", what, ws_bytes, L.total);
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 255) == 0, IKRL_ERR_ALIGNMENT,
               "%s: workspace must be 256-byte aligned", what);
  cudaStream_t s = as_stream(stream);
  char* w = reinterpret_cast<char*>(ws);
  int* err = reinterpret_cast<int*>(w + L.err_off);
  IKRL_CUDA(cudaMemsetAsync(err, 0, sizeof(int), s));

  CUtensorMap ta, tb, tb2;
  if ((rc = make_tmap(&ta, hidden, H, N, H, BM, "hidden"))) return rc;
  if ((rc = make_tmap(&tb, weight, H, V, H, BN, "weight"))) return rc;
  if ((rc = make_tmap(&tb2, weight, H, V, H, BN / 2, "weight"))) return rc;
  GemmParams p{};
  p.M = (int)N; p.N = V; p.K = H;
  p.ids = ids;
  p.id_offset = vocab_start;
  p.part_m = reinterpret_cast<float*>(w + L.pm_off);
  p.part_s = reinterpret_cast<float*>(w + L.ps_off);
  p.part_t = reinterpret_cast<float*>(w + L.pt_off);
  p.err = err;
  if (cache.slot != nullptr) {
    // Number the rows that get a cache slot (row order, at most cap of them).
    int* counts = reinterpret_cast<int*>(w + L.total);
    const int nb = (int)cdiv64(N, kCompactRows);
    cache_count_kernel<<<nb, kCompactThreads, 0, s>>>(cache.mask, ids, N, counts);
    if ((rc = check_launch("cache_count_kernel"))) return rc;
    cache_slot_kernel<<<nb, kCompactThreads, 0, s>>>(cache.mask, ids, N, counts, cache.cap, cache.slot);
    if ((rc = check_launch("cache_slot_kernel"))) return rc;
    p.slot = cache.slot;
    p.cache_q = cache.q;
    p.cache_m = cache.m;
    p.ld_cache = cdiv64(V, 64) * 64;
    p.n_mchunks = (int)cdiv64(V, 32);
  }
  CUtensorMap tq;
  if (cache.slot != nullptr && cache.cap > 0)
    if ((rc = make_store_tmap(&tq, cache.q, V, cache.cap, cdiv64(V, 64) * 64, "logit cache store"))) return rc;
  const int m_tiles = (int)cdiv64(N, BM);
  if (cache.slot != nullptr && cache.cap > 0) {
    if ((rc = launch_k1<EPI_LSE_CACHED, false, false>(ta, tb, ta, tb2, p, m_tiles, L.splits, s, &tq))) return rc;
  } else {
    if ((rc = launch_k1<EPI_LSE, false, false>(ta, tb, ta, tb2, p, m_tiles, L.splits, s))) return rc;
  }
  if (shard) {
    lse_shard_combine_kernel<<<(unsigned)cdiv64(N, 256), 256, 0, s>>>(p.part_m, p.part_s, p.part_t, ids, (int)N,
                                                                      vocab_start, V, p.part_sets, logp, lse, err);
    return check_launch("lse_shard_combine_kernel");
  }
  lse_combine_kernel<<<(unsigned)cdiv64(N, 256), 256, 0, s>>>(p.part_m, p.part_s, p.part_t, ids, (int)N, V,
                                                              p.part_sets, logp, lse, err);
  return check_launch("lse_combine_kernel");
}


// A dW over fewer rows than this is mostly its output: it takes the wide kernel with TMA stores.
constexpr int64_t kShortDw = 1024;

static int check_dweight_kind(const char* what, int32_t dweight_dtype, int32_t accumulate_dweight) {
  IKRL_REQUIRE(dweight_dtype == IKRL_DTYPE_F32 || dweight_dtype == IKRL_DTYPE_BF16, IKRL_ERR_UNSUPPORTED,
               "%s: dweight dtype %d unsupported", what, dweight_dtype);
  IKRL_REQUIRE(!(accumulate_dweight && dweight_dtype == IKRL_DTYPE_BF16), IKRL_ERR_UNSUPPORTED,
               "%s: accumulating into a bf16 dweight is not supported; use fp32", what);
  return IKRL_OK;
}

static int check_grad_alignment(const char* what, const void* dhidden, const void* dweight) {
  IKRL_REQUIRE(dweight == nullptr || (reinterpret_cast<uintptr_t>(dweight) & 15) == 0, IKRL_ERR_ALIGNMENT,
               "%s: dweight must be 16-byte aligned", what);
  IKRL_REQUIRE(dhidden == nullptr || (reinterpret_cast<uintptr_t>(dhidden) & 15) == 0, IKRL_ERR_ALIGNMENT,
               "%s: dhidden must be 16-byte aligned", what);
  return IKRL_OK;
}

// A bf16 dW of few rows: mostly its output, which leaves through TMA stores of the wide kernel, where that
// may run (two terms of 96 rows x 1024 for 151936 columns, 311 MB: 100 us; a plain fill of as much takes 88 us,
// and one term with stores from registers took 161 us).
static int launch_short_dw(const CUtensorMap& ta, const CUtensorMap& tb, GemmParams& p, void* dweight,
                           cudaStream_t s) {
  const int v_tiles = (int)cdiv64(p.M, BM);
  if (use_pairs() && tuning(IKRL_TUNE_WIDE) != 0) {
    CUtensorMap tc;
    const int rc = make_store_tmap(&tc, dweight, p.N, p.M, p.N, "dW store");
    if (rc) return rc;
    return launch_k1<EPI_STORE_TMA, true, true>(ta, tb, ta, tb, p, v_tiles, 0, s, &tc);
  }
  p.out_bf16 = reinterpret_cast<uint16_t*>(dweight); p.ld_bf16 = p.N;
  return launch_k1<EPI_STORE_BF16, true, true>(ta, tb, ta, tb, p, v_tiles, 0, s);
}

// The workspace of a RowRange.
static size_t row_range_bytes(int64_t N, int H, int V) {
  return 256 + 5 * align256((size_t)N * 4) + align256((size_t)N * H * 2) + align256((size_t)V * H * 2);
}
static RowRange row_range(char* w, int64_t N, int H) {
  RowRange R;
  const size_t n4 = align256((size_t)N * 4);
  R.top = reinterpret_cast<unsigned*>(w);
  R.dw_scale = reinterpret_cast<float*>(w) + 2;
  w += 256;
  R.e = reinterpret_cast<int*>(w);
  R.mul = reinterpret_cast<float*>(w + n4);
  R.gs = reinterpret_cast<float*>(w + 2 * n4);
  R.level = reinterpret_cast<float*>(w + 3 * n4);
  R.dh_scale = reinterpret_cast<float*>(w + 4 * n4);
  R.h = reinterpret_cast<uint16_t*>(w + 5 * n4);
  R.w = reinterpret_cast<uint16_t*>(w + 5 * n4 + align256((size_t)N * H * 2));
  return R;
}

// A row loss (row_dist.cuh) behind the LM head's backward: the state its forward left, and its level
// (the constant part of the gradient).
struct RowLossBwd {
  RowState st;
  int K;
  float c, level;
  bool all_cached;  // every row that is not kRowNone has a cache slot
};

// cache_slot / cache_q / cache_m: the logit cache a forward filled (all null: no cache).  Active
// rows with a slot take their dS from the cache; the others are recomputed by the dS GEMM.
// rl: null for log p(ids); otherwise the row loss whose gradient dlogp is, with ids and lse its
// state's row_ids and ref, and the workspace has a RowRange behind the layout's.
static int lmhead_bwd_impl(const char* what, const void* hidden, const void* weight, const int64_t* ids,
                           const float* lse, const float* dlogp, int64_t N, int32_t H, int32_t V, int64_t vocab_start,
                           int64_t chunk_rows, void* dhidden, void* dweight, int32_t dweight_dtype,
                           int32_t accumulate_dweight, void* ws, size_t ws_bytes, void* stream,
                           const int* cache_slot = nullptr, const uint16_t* cache_q = nullptr,
                           const float* cache_m = nullptr, const RowLossBwd* rl = nullptr) {
  int rc = check_common(hidden, weight, ids, N, H, V, what);
  if (rc) return rc;
  if ((rc = check_dweight_kind(what, dweight_dtype, accumulate_dweight))) return rc;
  if (N == 0) {  // no rows: dW is zero, or left as it is when accumulating
    if (dweight && !accumulate_dweight)
      IKRL_CUDA(cudaMemsetAsync(dweight, 0, (size_t)V * H * (dweight_dtype == IKRL_DTYPE_F32 ? 4 : 2),
                                as_stream(stream)));
    return clear_status_word(ws, ws_bytes, stream);
  }
  IKRL_REQUIRE(lse && dlogp && (dhidden || dweight), IKRL_ERR_INVALID_ARGUMENT,
               "%s: null pointer", what);
  const BwdLayout L = bwd_layout(N, H, V, chunk_rows, dweight_dtype, accumulate_dweight);
  const size_t ws_need = L.total + (rl ? row_range_bytes(N, H, V) : 0);
  IKRL_REQUIRE(ws != nullptr && ws_bytes >= ws_need, IKRL_ERR_WORKSPACE,
               "%s: workspace %zu < %zu bytes", what, ws_bytes, ws_need);
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 255) == 0, IKRL_ERR_ALIGNMENT,
               "%s: workspace must be 256-byte aligned", what);
  if ((rc = check_grad_alignment(what, dhidden, dweight))) return rc;
  cudaStream_t s = as_stream(stream);
  char* w = reinterpret_cast<char*>(ws);
  int* err = reinterpret_cast<int*>(w + L.err_off);
  uint16_t* dS = reinterpret_cast<uint16_t*>(w + L.ds_off);
  float* dw32 = L.need_dw32 ? reinterpret_cast<float*>(w + L.dw_off) : nullptr;
  IKRL_CUDA(cudaMemsetAsync(err, 0, sizeof(int), s));
  const int n_vt = (int)cdiv64(V, BN);
  int nsm = kNumSMs;
  {
    int dev = 0;
    IKRL_CUDA(cudaGetDevice(&dev));
    IKRL_CUDA(cudaDeviceGetAttribute(&nsm, cudaDevAttrMultiProcessorCount, dev));
  }

  // Rows the GEMMs run on: all N, or the compacted active rows.
  const uint16_t* hsrc = reinterpret_cast<const uint16_t*>(hidden);
  const int64_t* idsrc = ids;
  const float* lsesrc = lse;
  const float* gsrc = dlogp;
  int64_t Nw = N;
  uint16_t* dh_out = reinterpret_cast<uint16_t*>(dhidden);  // where the dH GEMMs write
  const int* pos = nullptr;                                  // set when dH must be scattered back
  const int* idx_c = nullptr;                                // compacted row -> row
  int64_t n_cached = 0;                                      // leading compacted rows whose dS is cached
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  IKRL_CUDA(cudaStreamIsCapturing(s, &cap));
  const bool skip_rows = skip_zero_rows_enabled() && cap == cudaStreamCaptureStatusNone && N <= INT32_MAX;
  if (skip_rows) {
    int* counts = reinterpret_cast<int*>(w + L.cnt_off);
    int64_t* n_act_d = reinterpret_cast<int64_t*>(w + L.nact_off);
    int* idx = reinterpret_cast<int*>(w + L.idx_off);
    int* posw = reinterpret_cast<int*>(w + L.pos_off);
    int64_t* ids_c = reinterpret_cast<int64_t*>(w + L.idc_off);
    float* lse_c = reinterpret_cast<float*>(w + L.lsec_off);
    float* g_c = reinterpret_cast<float*>(w + L.gc_off);
    uint16_t* h_c = reinterpret_cast<uint16_t*>(w + L.hc_off);
    const int nb = (int)cdiv64(N, kCompactRows);
    active_count_kernel<<<nb, kCompactThreads, 0, s>>>(dlogp, ids, cache_slot, N, counts);
    if ((rc = check_launch("active_count_kernel"))) return rc;
    compact_rows_kernel<<<nb, kCompactThreads, 0, s>>>(dlogp, ids, cache_slot, lse, N, counts, idx, posw, ids_c,
                                                        lse_c, g_c, n_act_d);
    if ((rc = check_launch("compact_rows_kernel"))) return rc;
    // The chunk plan depends on the active counts: read them back (one stream synchronisation).
    int64_t counts_h[2] = {0, 0};
    IKRL_CUDA(cudaMemcpyAsync(counts_h, n_act_d, 2 * sizeof(int64_t), cudaMemcpyDeviceToHost, s));
    IKRL_CUDA(cudaStreamSynchronize(s));
    const int64_t n_act = counts_h[0];
    n_cached = counts_h[1];
    IKRL_REQUIRE(n_act >= 0 && n_act <= N && n_cached >= 0 && n_cached <= n_act, IKRL_ERR_DEVICE,
                 "%s: bad active-row counts %lld, %lld", what, (long long)n_act, (long long)n_cached);
    if (n_act == 0) {
      if (dhidden) IKRL_CUDA(cudaMemsetAsync(dhidden, 0, (size_t)N * H * 2, s));
      if (dweight && !accumulate_dweight)
        IKRL_CUDA(cudaMemsetAsync(dweight, 0, (size_t)V * H * (dweight_dtype == IKRL_DTYPE_F32 ? 4 : 2), s));
      return IKRL_OK;
    }
    if (n_act < N || n_cached > 0) {  // cached rows come first, so the order differs from the rows'
      const int vpr = H / 8;
      const int gb = (int)std::min<int64_t>(cdiv64(n_act * vpr, 256), 148ll * 16);
      gather_rows_kernel<<<gb, 256, 0, s>>>(reinterpret_cast<const uint4*>(hidden), idx, n_act, vpr,
                                            reinterpret_cast<uint4*>(h_c));
      if ((rc = check_launch("gather_rows_kernel"))) return rc;
      hsrc = h_c; idsrc = ids_c; lsesrc = lse_c; gsrc = g_c; Nw = n_act; idx_c = idx;
      // dH of a chunk overwrites that chunk's gathered rows once dW has read them.
      if (dhidden) { dh_out = h_c; pos = posw; }
    }
  }

  const uint16_t* hw = hsrc;  // the dW operand
  RowRange R{};
  if (rl) {
    R = row_range(w + L.total, N, H);
    const int vpr = H / 8;
    IKRL_CUDA(cudaMemsetAsync(R.top, 0, 2 * sizeof(unsigned), s));
    const uint4* hv = reinterpret_cast<const uint4*>(hsrc);
    const int64_t nw = (int64_t)V * vpr;
    const unsigned wb = (unsigned)std::min<int64_t>(cdiv64(nw, 256), 148ll * 8);
    if (dhidden) {
      weight_range_kernel<<<wb, 256, 0, s>>>(reinterpret_cast<const uint4*>(weight), nw, R.top + 1);
      if ((rc = check_launch("weight_range_kernel"))) return rc;
    }
    row_range_kernel<<<(unsigned)cdiv64(Nw, 8), 256, 0, s>>>(dlogp, rl->st.row_ids, rl->st.coef, rl->st.cols, rl->st.grad,
                                                             rl->K, idx_c, Nw, rl->level, hv, vpr, R);
    if ((rc = check_launch("row_range_kernel"))) return rc;
    scale_rows_kernel<<<(unsigned)std::min<int64_t>(cdiv64(dweight ? Nw * vpr : Nw, 256), 148ll * 8), 256, 0, s>>>(
        dweight ? hv : nullptr, Nw, vpr, R);
    if ((rc = check_launch("scale_rows_kernel"))) return rc;
    if (dhidden) {
      scale_weight_kernel<<<wb, 256, 0, s>>>(reinterpret_cast<const uint4*>(weight), nw, R);
      if ((rc = check_launch("scale_weight_kernel"))) return rc;
    }
    gsrc = R.gs;
    hw = R.h;
  }

  const BwdLayout Lw = bwd_layout(Nw, H, V, chunk_rows, dweight_dtype, accumulate_dweight);
  const int64_t chunk = std::min(L.chunk, Lw.chunk);
  // Chunks: first the cached rows [0, n_cached), then the others, so every chunk takes its dS one
  // way (from the cache, or by the recompute GEMM).  Two such chunks need the fp32 accumulator of a
  // bf16 dweight; where the workspace has none (the rows fit one chunk), both kinds of rows share
  // one chunk: the cached ones are its first `cached`.
  struct Chunk {
    int64_t c0, rows, cached;
  };
  if (rl && rl->all_cached && cache_slot != nullptr) n_cached = Nw;
  std::vector<Chunk> chunks;
  if (n_cached > 0 && n_cached < Nw && Nw <= chunk && dweight && dweight_dtype == IKRL_DTYPE_BF16 && !L.need_dw32) {
    chunks.push_back({0, Nw, n_cached});
  } else {
    for (int seg = 0; seg < 2; ++seg) {
      const int64_t a0 = seg == 0 ? 0 : n_cached, a1 = seg == 0 ? n_cached : Nw;
      for (int64_t c0 = a0; c0 < a1; c0 += chunk) {
        const int64_t n = std::min<int64_t>(chunk, a1 - c0);
        chunks.push_back({c0, n, seg == 0 ? n : 0});
      }
    }
  }
  const int64_t nchunks = (int64_t)chunks.size();
  const bool use_dw32 = (dweight_dtype == IKRL_DTYPE_BF16) && nchunks > 1;

  CUtensorMap t_w_k, t_w_k2, t_w_mn;
  if ((rc = make_tmap(&t_w_k, weight, H, V, H, BN, "weight"))) return rc;
  if ((rc = make_tmap(&t_w_k2, weight, H, V, H, BN / 2, "weight"))) return rc;
  if ((rc = make_tmap(&t_w_mn, rl && dhidden ? (const void*)R.w : weight, H, V, H, 64, "weight^T"))) return rc;

  for (int64_t ci = 0; ci < nchunks; ++ci) {
    const int64_t c0 = chunks[ci].c0;
    const int64_t rows = chunks[ci].rows;
    const int m_tiles = (int)cdiv64(rows, BM);
    const uint16_t* hc = hw + c0 * H;
    // 1) dS = g * (onehot - softmax(h W^T)) for this chunk: from the logit cache, or recomputed
    const int64_t from_cache = chunks[ci].cached;  // leading rows of the chunk
    if (from_cache > 0 && rl) {
      const dim3 grid((unsigned)std::max<int64_t>(1, cdiv64(V / 8, 256 * kDsUnroll)),
                      (unsigned)std::min<int64_t>(from_cache, 65535));
      dtail_from_cache_kernel<false><<<grid, 256, 0, s>>>(
          cache_q, cache_m, L.lds, (int)cdiv64(V, 32), cache_slot, idx_c, dlogp,
          rl->st.row_ids, rl->st.ref, rl->st.coef, rl->st.cols, rl->st.grad, R.mul, rl->K, rl->level, rl->c, c0,
          from_cache, V, dS, L.lds);
      if ((rc = check_launch("dtail_from_cache_kernel"))) return rc;
    } else if (from_cache > 0) {
      const dim3 grid((unsigned)std::max<int64_t>(1, cdiv64(V / 8, 256 * kDsUnroll)),
                      (unsigned)std::min<int64_t>(from_cache, 65535));
      ds_from_cache_kernel<<<grid, 256, 0, s>>>(cache_q, cache_m, L.lds, (int)cdiv64(V, 32), cache_slot, idx_c,
                                                idsrc, lsesrc, gsrc, c0, from_cache, V, vocab_start, dS, L.lds);
      if ((rc = check_launch("ds_from_cache_kernel"))) return rc;
    }
    if (from_cache < rows) {
      const int64_t r0 = c0 + from_cache, nr = rows - from_cache;
      uint16_t* dS_r = dS + from_cache * L.lds;
      CUtensorMap ta, tds;
      if ((rc = make_tmap(&ta, hsrc + r0 * H, H, nr, H, BM, "hidden chunk"))) return rc;
      if ((rc = make_store_tmap(&tds, dS_r, V, nr, L.lds, "dS store"))) return rc;
      GemmParams p{};
      p.M = (int)nr; p.N = V; p.K = H;
      const int nr_tiles = (int)cdiv64(nr, BM);
      const int sp = choose_splits(nr_tiles, n_vt, H);
      p.ids = idsrc + r0; p.lse = lsesrc + r0; p.g = gsrc + r0;
      p.id_offset = vocab_start;
      p.out_bf16 = dS_r; p.ld_bf16 = L.lds;
      p.err = err;
      if (rl) {
        p.level = R.level + r0;
        p.c = rl->c;
        p.f16 = 1;
        if ((rc = launch_k1<EPI_DTAIL, false, false>(ta, t_w_k, ta, t_w_k2, p, nr_tiles, sp, s, &tds))) return rc;
      } else {
        if ((rc = launch_k1<EPI_DLOGITS, false, false>(ta, t_w_k, ta, t_w_k2, p, nr_tiles, sp, s, &tds))) return rc;
      }
    }
    if (rl && from_cache < rows) {
      const int64_t n = rows - from_cache;
      ds_entries_kernel<false><<<(unsigned)cdiv64(n * rl->K, 256), 256, 0, s>>>(
          dlogp, rl->st.cols, rl->st.grad, R.mul, rl->K, idx_c, c0 + from_cache, n, dS + from_cache * L.lds, L.lds);
      if ((rc = check_launch("ds_entries_kernel"))) return rc;
    }
    // 2) dW (+)= dS^T h[chunk]
    if (dweight) {
      CUtensorMap ta, tb;
      if ((rc = make_tmap(&ta, dS, V, rows, L.lds, 64, "dS^T"))) return rc;
      if ((rc = make_tmap(&tb, hc, H, rows, H, 64, "hidden chunk^T"))) return rc;
      GemmParams p{};
      p.M = V; p.N = H; p.K = (int)rows;
      p.err = err;
      if (rl) { p.f16 = 1; p.out_scale = R.dw_scale; }
      const int v_tiles = (int)cdiv64(V, BM);
      const bool last = ci == nchunks - 1;
      if (dweight_dtype == IKRL_DTYPE_BF16 && !use_dw32 && rl && rows < kShortDw) {
        if ((rc = launch_short_dw(ta, tb, p, dweight, s))) return rc;
      } else if (dweight_dtype == IKRL_DTYPE_BF16 && !use_dw32) {
        p.out_bf16 = reinterpret_cast<uint16_t*>(dweight); p.ld_bf16 = H;
        if ((rc = launch_k1<EPI_STORE_BF16, true, true>(ta, tb, ta, tb, p, v_tiles, 0, s))) return rc;
      } else {
        if (dweight_dtype == IKRL_DTYPE_F32) {
          p.out_f32 = reinterpret_cast<float*>(dweight);
          p.f32_mode = (ci == 0 && !accumulate_dweight) ? F32_STORE : F32_ADD;
        } else {
          p.out_f32 = dw32;
          p.out_bf16 = reinterpret_cast<uint16_t*>(dweight); p.ld_bf16 = H;
          p.f32_mode = last ? F32_ADD_TO_BF16 : (ci == 0 ? F32_STORE : F32_ADD);
        }
        p.ld_f32 = H;
        if ((rc = launch_k1<EPI_F32, true, true>(ta, tb, ta, tb, p, v_tiles, 0, s))) return rc;
      }
    }
    // 3) dH[chunk] = dS W, whole or as K-range partials summed afterwards
    if (dhidden) {
      CUtensorMap ta;
      if ((rc = make_tmap(&ta, dS, V, rows, L.lds, BM, "dS"))) return rc;
      GemmParams p{};
      p.M = (int)rows; p.N = H; p.K = V;
      p.err = err;
      if (rl) { p.f16 = 1; p.out_scale = R.dh_scale + c0; p.scale_rows = 1; }
      const int ks = dh_split_k(m_tiles, H, V, rows, L.part_elems, nsm, rl != nullptr);
      if (ks > 1) {
        float* part = reinterpret_cast<float*>(w + L.part_off);
        p.out_f32 = part; p.ld_f32 = H; p.f32_mode = F32_STORE;
        p.ksplits = ks; p.ks_stride = rows * H;
        if ((rc = launch_k1<EPI_F32, false, true>(ta, t_w_mn, ta, t_w_mn, p, m_tiles, 0, s))) return rc;
        const int64_t n4 = rows * H / 4;
        const int gb = (int)std::min<int64_t>(cdiv64(n4, 256), 148ll * 8);
        splitk_sum_kernel<<<gb, 256, 0, s>>>(reinterpret_cast<const float4*>(part), n4, ks,
                                             reinterpret_cast<uint2*>(dh_out + c0 * H));
        if ((rc = check_launch("splitk_sum_kernel"))) return rc;
      } else {
        p.out_bf16 = dh_out + c0 * H; p.ld_bf16 = H;
        if ((rc = launch_k1<EPI_STORE_BF16, false, true>(ta, t_w_mn, ta, t_w_mn, p, m_tiles, 0, s))) return rc;
      }
    }
  }
  if (pos != nullptr) {
    const int vpr = H / 8;
    const int gb = (int)std::min<int64_t>(cdiv64(N * vpr, 256), 148ll * 16);
    scatter_rows_kernel<<<gb, 256, 0, s>>>(reinterpret_cast<const uint4*>(dh_out), pos, N, vpr,
                                           reinterpret_cast<uint4*>(dhidden));
    if ((rc = check_launch("scatter_rows_kernel"))) return rc;
  }
  return IKRL_OK;
}

// The logit cache of a row loss: slots 0, 1, ... go to the rows that count, in row order, while there
// are any (rows = 0: no cache).
struct RowCacheArgs {
  int64_t rows;
  int* slot;
  uint16_t* q;
  float* m;
};

static int check_row_cache(const char* what, int64_t N, int V, const RowCacheArgs& c) {
  IKRL_REQUIRE(c.rows >= 0, IKRL_ERR_INVALID_ARGUMENT, "%s: cache_rows %lld < 0", what, (long long)c.rows);
  if (c.rows == 0 || N == 0) return IKRL_OK;
  IKRL_REQUIRE(V % 8 == 0, IKRL_ERR_UNSUPPORTED, "%s: the logit cache needs V (%d) to be a multiple of 8", what, V);
  IKRL_REQUIRE(c.slot && c.q && c.m, IKRL_ERR_INVALID_ARGUMENT, "%s: null cache pointer", what);
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(c.q) & 15) == 0 && (reinterpret_cast<uintptr_t>(c.m) & 3) == 0,
               IKRL_ERR_ALIGNMENT, "%s: cache_q must be 16-byte and cache_m 4-byte aligned", what);
  return IKRL_OK;
}

// Forward of a row loss through the LM head: the rows' entries, the rows that count gathered, the GEMM with
// the TAIL epilogue, the losses.
static int lmhead_row_loss_fwd(const char* what, const void* hidden, const void* weight, const int64_t* tids,
                               const float* tlp, int64_t N, int32_t H, int32_t V, int32_t K, const RowLossParams& P,
                               float* loss, void* state, size_t state_bytes, const RowCacheArgs& cache, void* ws,
                               size_t ws_bytes, void* stream) {
  int rc = check_common(hidden, weight, tids, N, H, V, what);
  if (rc) return rc;
  if (N == 0) return clear_status_word(ws, ws_bytes, stream);
  IKRL_REQUIRE(loss != nullptr, IKRL_ERR_INVALID_ARGUMENT, "%s: output is NULL", what);
  IKRL_REQUIRE(state != nullptr && state_bytes >= row_state_bytes(N, K), IKRL_ERR_WORKSPACE,
               "%s: state %zu < %zu bytes", what, state_bytes, row_state_bytes(N, K));
  const RowLossFwdLayout L = row_loss_fwd_layout(N, H, V);
  IKRL_REQUIRE(ws != nullptr && ws_bytes >= L.total, IKRL_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", what,
               ws_bytes, L.total);
  IKRL_REQUIRE(((reinterpret_cast<uintptr_t>(ws) | reinterpret_cast<uintptr_t>(state)) & 255) == 0,
               IKRL_ERR_ALIGNMENT, "%s: workspace and state must be 256-byte aligned", what);
  IKRL_REQUIRE(((reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(weight)) & 15) == 0,
               IKRL_ERR_ALIGNMENT, "%s: hidden and weight must be 16-byte aligned", what);
  if ((rc = check_row_cache(what, N, V, cache))) return rc;
  cudaStream_t s = as_stream(stream);
  const RowState st = row_state(state, N, K);
  char* w = reinterpret_cast<char*>(ws);
  int* err = reinterpret_cast<int*>(w);
  if ((rc = launch_row_entries(tids, tlp, N, K, P, st, s, err))) return rc;
  const int vpr = H / 8;
  GemmParams p{};
  const bool exact_tops = H >= kExactTopsHidden;
  if (P.loss == ROW_XENT && !exact_tops) {
    p.xk = st.xk;
  } else {
    IKRL_REQUIRE(cdiv64(N * K, 8) <= 0x7fffffffLL, IKRL_ERR_UNSUPPORTED, "%s: %lld rows of %d entries", what,
                 (long long)N, K);
    entry_logits_kernel<<<(unsigned)cdiv64(N * K, 8), 256, 0, s>>>(reinterpret_cast<const uint4*>(hidden),
                                                                   reinterpret_cast<const uint4*>(weight), st.cols,
                                                                   N * K, K, vpr, st.xk);
    if ((rc = check_launch("entry_logits_kernel"))) return rc;
  }

  p.M = (int)N; p.N = V; p.K = H;
  p.part_m = reinterpret_cast<float*>(w + L.pm_off);
  p.part_s = reinterpret_cast<float*>(w + L.ps_off);
  p.part_c = exact_tops ? reinterpret_cast<int*>(w + L.pc_off) : nullptr;
  p.part_cap = L.sets;
  p.part_x = P.loss == ROW_XENT && P.smoothing != 0.f ? reinterpret_cast<float*>(w + L.px_off) : nullptr;
  p.err = err;
  p.c = P.c;
  p.cols = st.cols;
  p.n_cols = K;
  const void* rows_in = hidden;
  const int* pos = nullptr;
  // Without gathering a cache is used when it holds every row, and row r takes slot r: nothing to number.
  const bool cached = L.gather ? cache.rows > 0 : cache.rows >= N;
  if (L.gather) {
    int* counts = reinterpret_cast<int*>(w + L.counts_off);
    int* count = reinterpret_cast<int*>(w + L.count_off);
    int* posw = reinterpret_cast<int*>(w + L.pos_off);
    int* idx = reinterpret_cast<int*>(w + L.idx_off);
    const int nb = (int)cdiv64(N, kCompactRows);
    cache_count_kernel<<<nb, kCompactThreads, 0, s>>>(nullptr, st.row_ids, N, counts);
    if ((rc = check_launch("cache_count_kernel"))) return rc;
    cache_slot_kernel<<<nb, kCompactThreads, 0, s>>>(nullptr, st.row_ids, N, counts, N, posw);
    if ((rc = check_launch("cache_slot_kernel"))) return rc;
    int dev = 0, nsm = kNumSMs;
    IKRL_CUDA(cudaGetDevice(&dev));
    IKRL_CUDA(cudaDeviceGetAttribute(&nsm, cudaDevAttrMultiProcessorCount, dev));
    const K1Plan pl = plan_k1(EPI_TAIL, cdiv64(N, BM), V, H, L.splits, nsm);
    LiveSplit ls{pl.n_tiles, pl.tiles_per_split, pl.splits, 0, 0, std::max(1, nsm / 2), pl.kind == 2 ? kWideGroups : 1};
    if (pl.kind != 0 && persistent_pairs() && balance_splits_enabled()) {
      ls.least = std::min(L.splits, pl.n_tiles);
      ls.most = std::min(kBalanceMost * L.splits, pl.n_tiles);
    }
    IKRL_REQUIRE(std::max(ls.most, ls.splits) * ls.groups <= L.sets, IKRL_ERR_WORKSPACE,
                 "%s: %d column ranges of %d groups, room for %d sets", what, std::max(ls.most, ls.splits), ls.groups,
                 L.sets);
    row_index_kernel<<<(unsigned)cdiv64(N, 256), 256, 0, s>>>(posw, N, cache.rows, idx, cached ? cache.slot : nullptr,
                                                              counts, nb, ls, count);
    if ((rc = check_launch("row_index_kernel"))) return rc;
    uint4* hc = reinterpret_cast<uint4*>(w + L.hc_off);
    gather_live_rows_kernel<<<(unsigned)std::min<int64_t>(cdiv64(N * vpr, 256), 148ll * 16), 256, 0, s>>>(
        reinterpret_cast<const uint4*>(hidden), idx, count, vpr, hc);
    if ((rc = check_launch("gather_live_rows_kernel"))) return rc;
    rows_in = hc;
    pos = posw;
    p.m_dev = count;
    p.row_idx = idx;
  }
  if (cached) {
    p.cache_cap = cache.rows;
    p.cache_q = cache.q;
    p.cache_m = cache.m;
    p.ld_cache = cdiv64(V, 64) * 64;
    p.n_mchunks = (int)cdiv64(V, 32);
  }
  CUtensorMap ta, tb, tb2, tq;
  if ((rc = make_tmap(&ta, rows_in, H, N, H, BM, "hidden"))) return rc;
  if ((rc = make_tmap(&tb, weight, H, V, H, BN, "weight"))) return rc;
  if ((rc = make_tmap(&tb2, weight, H, V, H, BN / 2, "weight"))) return rc;
  const int m_tiles = (int)cdiv64(N, BM);
  if (cached) {
    if ((rc = make_store_tmap(&tq, cache.q, V, cache.rows, p.ld_cache, "logit cache store"))) return rc;
    if ((rc = launch_k1<EPI_TAIL_CACHED, false, false>(ta, tb, ta, tb2, p, m_tiles, L.splits, s, &tq))) return rc;
  } else {
    if ((rc = launch_k1<EPI_TAIL, false, false>(ta, tb, ta, tb2, p, m_tiles, L.splits, s))) return rc;
  }
  const int* sets_dev = p.m_dev ? p.m_dev + LIVE_SETS : nullptr;
  if (exact_tops) {
    const bool wide_rows = row_takes_a_block(p.part_sets, N);
    auto kern = wide_rows ? exact_tops_kernel<4> : exact_tops_kernel<1>;
    kern<<<(unsigned)(wide_rows ? N : cdiv64(N, 4)), 128, 0, s>>>(
        reinterpret_cast<const uint4*>(hidden), reinterpret_cast<const uint4*>(weight), vpr, p.part_m, p.part_c, p.part_s,
        p.part_sets, sets_dev, pos, st.row_ids, st.xk, st.cols, K, N, V, P.c, err);
    if ((rc = check_launch("exact_tops_kernel"))) return rc;
  }
  return launch_row_losses(p.part_m, p.part_s, p.part_x, p.part_sets, sets_dev, pos, N, K, P, st, loss, err, s);
}

// Backward of a row loss of few rows (row_loss_dense), all of them in one chunk, without the
// compaction and its host synchronisation.  dS is held in two terms, hi = bf16(d) and lo = bf16(d - hi),
// stacked as 2N rows: dW = [hi; lo]^T [h; h], dH = hi W + lo W.  With few rows a sum over the rows averages
// little of dS's rounding away, and one term alone would leave dW with up to twice the error that its own
// rounding to bf16 has; the second term costs K blocks of a dW that is bound by writing [V, H], and rows of a
// tile of dH that N <= 128 left empty.
struct FewLayout {
  size_t ds_off, h_off, gs_off, level_off, part_off, total;
  int64_t lds, part_sets;
};
static FewLayout few_layout(int64_t N, int H, int V) {
  FewLayout L;
  L.lds = cdiv64(V, 64) * 64;
  L.part_sets = std::max<int64_t>(1, kNumSMs / 2 / (cdiv64(H, WN) * cdiv64(2 * N, 2 * BM)));
  size_t o = 256;  // the error word
  L.ds_off = o; o += align256((size_t)2 * N * L.lds * 2);
  L.h_off = o; o += align256((size_t)2 * N * H * 2);
  L.gs_off = o; o += align256((size_t)N * 4);
  L.level_off = o; o += align256((size_t)N * 4);
  L.part_off = o; o += align256((size_t)L.part_sets * 2 * N * H * 4);
  L.total = o;
  return L;
}

// dweight's checks; the workspace is the caller's to check.
static int lmhead_row_loss_bwd_few(const char* what, const void* hidden, const void* weight, const float* dloss,
                                   int64_t N, int H, int V, const RowLossBwd& rl, void* dhidden, void* dweight,
                                   int32_t dweight_dtype, int32_t accumulate_dweight, const RowCacheArgs& cache,
                                   void* ws, void* stream) {
  int rc = check_common(hidden, weight, rl.st.row_ids, N, H, V, what);
  if (rc) return rc;
  if ((rc = check_dweight_kind(what, dweight_dtype, accumulate_dweight))) return rc;
  if ((rc = check_grad_alignment(what, dhidden, dweight))) return rc;
  IKRL_REQUIRE(dloss && (dhidden || dweight), IKRL_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 255) == 0, IKRL_ERR_ALIGNMENT,
               "%s: workspace must be 256-byte aligned", what);
  cudaStream_t s = as_stream(stream);
  const FewLayout L = few_layout(N, H, V);
  char* w = reinterpret_cast<char*>(ws);
  int* err = reinterpret_cast<int*>(w);
  uint16_t* ds = reinterpret_cast<uint16_t*>(w + L.ds_off);
  const bool cached = cache.rows >= N;
  float* gs = cached ? nullptr : reinterpret_cast<float*>(w + L.gs_off);
  float* level = reinterpret_cast<float*>(w + L.level_off);
  uint4* h2 = dweight ? reinterpret_cast<uint4*>(w + L.h_off) : nullptr;
  few_rows_kernel<<<(unsigned)N, 128, 0, s>>>(reinterpret_cast<const uint4*>(hidden), H / 8, h2, dloss, rl.st.row_ids,
                                              rl.st.coef, rl.level, gs, level, err);
  if ((rc = check_launch("few_rows_kernel"))) return rc;
  // 1) dS, from the forward's numerators or by the GEMM again
  if (cached) {
    const dim3 grid((unsigned)std::max<int64_t>(1, cdiv64(V / 8, 256 * kDsUnroll)), (unsigned)N);
    dtail_from_cache_kernel<true><<<grid, 256, 0, s>>>(cache.q, cache.m, L.lds, (int)cdiv64(V, 32), nullptr, nullptr,
                                                       dloss, rl.st.row_ids, rl.st.ref, rl.st.coef, rl.st.cols,
                                                       rl.st.grad, nullptr, rl.K, rl.level, rl.c, 0, N, V, ds, L.lds);
    if ((rc = check_launch("dtail_from_cache_kernel"))) return rc;
  } else {
    CUtensorMap ta, tb, tb2, tds;
    if ((rc = make_tmap(&ta, hidden, H, N, H, BM, "hidden"))) return rc;
    if ((rc = make_tmap(&tb, weight, H, V, H, BN, "weight"))) return rc;
    if ((rc = make_tmap(&tb2, weight, H, V, H, BN / 2, "weight"))) return rc;
    if ((rc = make_store_tmap(&tds, ds, V, N, L.lds, "dS store"))) return rc;
    GemmParams p{};
    p.M = (int)N; p.N = V; p.K = H;
    p.ids = rl.st.row_ids; p.lse = rl.st.ref; p.g = gs; p.level = level; p.c = rl.c;
    p.out_bf16 = ds; p.ld_bf16 = L.lds; p.out_lo = ds + N * L.lds;
    p.err = err;
    const int m_tiles = (int)cdiv64(N, BM);
    const int sp = choose_splits(m_tiles, (int)cdiv64(V, BN), H);
    if ((rc = launch_k1<EPI_DTAIL, false, false>(ta, tb, ta, tb2, p, m_tiles, sp, s, &tds))) return rc;
    ds_entries_kernel<true><<<(unsigned)cdiv64(N * rl.K, 256), 256, 0, s>>>(dloss, rl.st.cols, rl.st.grad, nullptr, rl.K,
                                                                            nullptr, 0, N, ds, L.lds);
    if ((rc = check_launch("ds_entries_kernel"))) return rc;
  }
  // 2) dW (+)= [hi; lo]^T [h; h]
  if (dweight) {
    CUtensorMap ta, tb;
    if ((rc = make_tmap(&ta, ds, V, 2 * N, L.lds, 64, "dS^T"))) return rc;
    if ((rc = make_tmap(&tb, h2, H, 2 * N, H, 64, "hidden^T"))) return rc;
    GemmParams p{};
    p.M = V; p.N = H; p.K = (int)(2 * N);
    p.err = err;
    if (dweight_dtype == IKRL_DTYPE_BF16) {
      if ((rc = launch_short_dw(ta, tb, p, dweight, s))) return rc;
    } else {
      p.out_f32 = reinterpret_cast<float*>(dweight); p.ld_f32 = H;
      p.f32_mode = accumulate_dweight ? F32_ADD : F32_STORE;
      if ((rc = launch_k1<EPI_F32, true, true>(ta, tb, ta, tb, p, (int)cdiv64(V, BM), 0, s))) return rc;
    }
  }
  // 3) dH = hi W + lo W: K ranges as many as keep every pair busy, each at least 16 K blocks (the rule for
  // more rows stops at 16 ranges, which leaves more than half of the pairs idle at H = 1024)
  if (dhidden) {
    const int64_t rows = 2 * N;
    CUtensorMap ta, tb;
    if ((rc = make_tmap(&ta, ds, V, rows, L.lds, BM, "dS"))) return rc;
    if ((rc = make_tmap(&tb, weight, H, V, H, 64, "weight^T"))) return rc;
    int64_t ks = 1;
    if (tuning(IKRL_TUNE_DH_SPLIT_K) < 0 && use_pairs() && use_wide(V) && persistent_pairs())
      ks = std::max<int64_t>(1, std::min(L.part_sets, cdiv64(V, BK) / 16));
    float* part = reinterpret_cast<float*>(w + L.part_off);
    GemmParams p{};
    p.M = (int)rows; p.N = H; p.K = V;
    p.err = err;
    p.out_f32 = part; p.ld_f32 = H; p.f32_mode = F32_STORE;
    if (ks > 1) { p.ksplits = (int)ks; p.ks_stride = rows * H; }
    if ((rc = launch_k1<EPI_F32, false, true>(ta, tb, ta, tb, p, (int)cdiv64(rows, BM), 0, s))) return rc;
    const int64_t n4 = N * H / 4;
    two_term_sum_kernel<<<(unsigned)cdiv64(n4, kTermSumGroups), 4 * kTermSumGroups, 0, s>>>(
        reinterpret_cast<const float4*>(part), n4, 2 * (int)ks, reinterpret_cast<uint2*>(dhidden));
    if ((rc = check_launch("two_term_sum_kernel"))) return rc;
  }
  return IKRL_OK;
}

static int lmhead_row_loss_bwd(const char* what, const void* hidden, const void* weight, int64_t N, int32_t H,
                               int32_t V, int32_t K, const RowLossParams& P, const void* state, size_t state_bytes,
                               const float* dloss, int64_t chunk_rows, void* dhidden, void* dweight,
                               int32_t dweight_dtype, int32_t accumulate_dweight, const RowCacheArgs& cache, void* ws,
                               size_t ws_bytes, void* stream) {
  int rc = check_row_cache(what, N, V, cache);
  if (rc) return rc;
  RowLossBwd rl{};
  if (N > 0) {
    IKRL_REQUIRE(state != nullptr && state_bytes >= row_state_bytes(N, K), IKRL_ERR_WORKSPACE,
                 "%s: state %zu < %zu bytes", what, state_bytes, row_state_bytes(N, K));
    IKRL_REQUIRE((reinterpret_cast<uintptr_t>(state) & 255) == 0, IKRL_ERR_ALIGNMENT,
                 "%s: state must be 256-byte aligned", what);
    const size_t need = ikrl_lmhead_row_loss_bwd_workspace_bytes(N, H, V, chunk_rows, dweight_dtype,
                                                                 accumulate_dweight);
    IKRL_REQUIRE(ws != nullptr && ws_bytes >= need, IKRL_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", what,
                 ws_bytes, need);
    IKRL_REQUIRE(((reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(weight)) & 15) == 0,
                 IKRL_ERR_ALIGNMENT, "%s: hidden and weight must be 16-byte aligned", what);
    rl.st = row_state(const_cast<void*>(state), N, K);
  }
  rl.K = K;
  rl.c = P.c;
  rl.level = P.loss == ROW_XENT ? -P.smoothing / (float)V : 0.f;
  rl.all_cached = cache.rows >= N;
  if (N > 0 && row_loss_dense(N, H, V))
    return lmhead_row_loss_bwd_few(what, hidden, weight, dloss, N, H, V, rl, dhidden, dweight, dweight_dtype,
                                   accumulate_dweight, cache, ws, stream);
  const bool cached = cache.rows > 0;
  return lmhead_bwd_impl(what, hidden, weight, rl.st.row_ids, rl.st.ref, dloss, N, H, V, 0, chunk_rows, dhidden,
                         dweight, dweight_dtype, accumulate_dweight, ws, ws_bytes, stream,
                         cached ? cache.slot : nullptr, cached ? cache.q : nullptr, cached ? cache.m : nullptr, &rl);
}


extern "C" {

size_t ikrl_lmhead_row_loss_fwd_workspace_bytes(int64_t N, int32_t H, int32_t V) {
  if (N <= 0 || H <= 0 || V <= 0) return 256;
  return row_loss_fwd_layout(N, H, V).total;
}

size_t ikrl_lmhead_row_loss_bwd_workspace_bytes(int64_t N, int32_t H, int32_t V, int64_t chunk_rows,
                                                int32_t dweight_dtype, int32_t accumulate_dweight) {
  if (N <= 0 || H <= 0 || V <= 0) return 256;
  if (row_loss_dense(N, H, V)) return few_layout(N, H, V).total;
  return bwd_layout(N, H, V, chunk_rows, dweight_dtype, accumulate_dweight).total + row_range_bytes(N, H, V);
}

int ikrl_lmhead_distill_fwd(const void* hidden, const void* weight, const int64_t* teacher_ids,
                            const float* teacher_logp, int64_t N, int32_t H, int32_t V, int32_t K,
                            const ikrl_distill_params* params, float* loss, void* state, size_t state_bytes,
                            int64_t cache_rows, int32_t* cache_slot, void* cache_q, float* cache_m, void* ws,
                            size_t ws_bytes, void* stream) {
  clear_error();
  const char* what = "ikrl_lmhead_distill_fwd";
  RowLossParams P;
  int rc = distill_params(what, params, V, K, &P);
  if (rc) return rc;
  IKRL_REQUIRE(N <= 0 || teacher_logp, IKRL_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  return lmhead_row_loss_fwd(what, hidden, weight, teacher_ids, teacher_logp, N, H, V, K, P, loss, state, state_bytes,
                             {cache_rows, cache_slot, reinterpret_cast<uint16_t*>(cache_q), cache_m}, ws, ws_bytes,
                             stream);
}

int ikrl_lmhead_distill_bwd(const void* hidden, const void* weight, int64_t N, int32_t H, int32_t V, int32_t K,
                            const ikrl_distill_params* params, const void* state, size_t state_bytes,
                            const float* dloss, int64_t chunk_rows, void* dhidden, void* dweight,
                            int32_t dweight_dtype, int32_t accumulate_dweight, int64_t cache_rows,
                            const int32_t* cache_slot, const void* cache_q, const float* cache_m, void* ws,
                            size_t ws_bytes, void* stream) {
  clear_error();
  const char* what = "ikrl_lmhead_distill_bwd";
  RowLossParams P;
  int rc = distill_params(what, params, V, K, &P);
  if (rc) return rc;
  return lmhead_row_loss_bwd(what, hidden, weight, N, H, V, K, P, state, state_bytes, dloss, chunk_rows, dhidden,
                             dweight, dweight_dtype, accumulate_dweight,
                             {cache_rows, const_cast<int32_t*>(cache_slot),
                              reinterpret_cast<uint16_t*>(const_cast<void*>(cache_q)), const_cast<float*>(cache_m)},
                             ws, ws_bytes, stream);
}

int ikrl_lmhead_cross_entropy_fwd(const void* hidden, const void* weight, const int64_t* targets, int64_t N,
                                  int32_t H, int32_t V, float label_smoothing, float z_loss, float* loss, void* state,
                                  size_t state_bytes, int64_t cache_rows, int32_t* cache_slot, void* cache_q,
                                  float* cache_m, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  const char* what = "ikrl_lmhead_cross_entropy_fwd";
  RowLossParams P;
  int rc = xent_params(what, label_smoothing, z_loss, V, &P);
  if (rc) return rc;
  return lmhead_row_loss_fwd(what, hidden, weight, targets, nullptr, N, H, V, 1, P, loss, state, state_bytes,
                             {cache_rows, cache_slot, reinterpret_cast<uint16_t*>(cache_q), cache_m}, ws, ws_bytes,
                             stream);
}

int ikrl_lmhead_cross_entropy_bwd(const void* hidden, const void* weight, int64_t N, int32_t H, int32_t V,
                                  float label_smoothing, float z_loss, const void* state, size_t state_bytes,
                                  const float* dloss, int64_t chunk_rows, void* dhidden, void* dweight,
                                  int32_t dweight_dtype, int32_t accumulate_dweight, int64_t cache_rows,
                                  const int32_t* cache_slot, const void* cache_q, const float* cache_m, void* ws,
                                  size_t ws_bytes, void* stream) {
  clear_error();
  const char* what = "ikrl_lmhead_cross_entropy_bwd";
  RowLossParams P;
  int rc = xent_params(what, label_smoothing, z_loss, V, &P);
  if (rc) return rc;
  return lmhead_row_loss_bwd(what, hidden, weight, N, H, V, 1, P, state, state_bytes, dloss, chunk_rows, dhidden,
                             dweight, dweight_dtype, accumulate_dweight,
                             {cache_rows, const_cast<int32_t*>(cache_slot),
                              reinterpret_cast<uint16_t*>(const_cast<void*>(cache_q)), const_cast<float*>(cache_m)},
                             ws, ws_bytes, stream);
}

size_t ikrl_lmhead_fwd_workspace_bytes(int64_t N, int32_t H, int32_t V) {
  if (N <= 0 || H <= 0 || V <= 0) return 256;
  return fwd_layout(N, H, V).total;
}

int ikrl_lmhead_logprob_fwd(const void* hidden, const void* weight, const int64_t* ids, int64_t N, int32_t H,
                            int32_t V, float* logp, float* lse, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  return lmhead_fwd_impl("ikrl_lmhead_logprob_fwd", hidden, weight, ids, N, H, V, 0, false, logp, lse, ws, ws_bytes,
                         stream);
}

int ikrl_lmhead_shard_fwd(const void* hidden, const void* weight_shard, const int64_t* ids, int64_t N, int32_t H,
                          int32_t V_shard, int64_t vocab_start, float* tlogit, float* lse_shard, void* ws,
                          size_t ws_bytes, void* stream) {
  clear_error();
  IKRL_REQUIRE(vocab_start >= 0, IKRL_ERR_INVALID_ARGUMENT, "ikrl_lmhead_shard_fwd: vocab_start %lld < 0",
               (long long)vocab_start);
  IKRL_REQUIRE(N == 0 || lse_shard != nullptr, IKRL_ERR_INVALID_ARGUMENT, "ikrl_lmhead_shard_fwd: lse_shard is NULL");
  return lmhead_fwd_impl("ikrl_lmhead_shard_fwd", hidden, weight_shard, ids, N, H, V_shard, vocab_start, true, tlogit,
                         lse_shard, ws, ws_bytes, stream);
}

int ikrl_vocab_parallel_combine(const float* parts, const int64_t* ids, int64_t N, int32_t P, int64_t V_total,
                                float* logp, float* lse, void* stream) {
  clear_error();
  IKRL_REQUIRE(N >= 0 && P >= 1 && V_total > 0, IKRL_ERR_INVALID_ARGUMENT,
               "ikrl_vocab_parallel_combine: bad sizes N=%lld P=%d V=%lld", (long long)N, P, (long long)V_total);
  if (N == 0) return IKRL_OK;
  IKRL_REQUIRE(parts && ids && logp, IKRL_ERR_INVALID_ARGUMENT, "ikrl_vocab_parallel_combine: null pointer");
  vocab_parallel_combine_kernel<<<(unsigned)cdiv64(N, 256), 256, 0, as_stream(stream)>>>(parts, ids, N, P, V_total,
                                                                                        logp, lse);
  return check_launch("vocab_parallel_combine_kernel");
}

size_t ikrl_lmhead_bwd_workspace_bytes(int64_t N, int32_t H, int32_t V, int64_t chunk_rows, int32_t dweight_dtype,
                                       int32_t accumulate_dweight) {
  if (N <= 0 || H <= 0 || V <= 0) return 256;
  return bwd_layout(N, H, V, chunk_rows, dweight_dtype, accumulate_dweight).total;
}

int ikrl_lmhead_logprob_bwd(const void* hidden, const void* weight, const int64_t* ids, const float* lse,
                            const float* dlogp, int64_t N, int32_t H, int32_t V, int64_t chunk_rows, void* dhidden,
                            void* dweight, int32_t dweight_dtype, int32_t accumulate_dweight, void* ws,
                            size_t ws_bytes, void* stream) {
  clear_error();
  return lmhead_bwd_impl("ikrl_lmhead_logprob_bwd", hidden, weight, ids, lse, dlogp, N, H, V, 0, chunk_rows, dhidden,
                         dweight, dweight_dtype, accumulate_dweight, ws, ws_bytes, stream);
}

int ikrl_lmhead_cache_row_elems(int32_t V, int64_t* q_elems, int64_t* m_elems) {
  clear_error();
  IKRL_REQUIRE(V > 0 && q_elems && m_elems, IKRL_ERR_INVALID_ARGUMENT, "ikrl_lmhead_cache_row_elems: bad arguments");
  *q_elems = cdiv64(V, 64) * 64;
  *m_elems = cdiv64(V, 32);
  return IKRL_OK;
}

size_t ikrl_lmhead_cache_fwd_workspace_bytes(int64_t N, int32_t H, int32_t V) {
  if (N <= 0 || H <= 0 || V <= 0) return 256;
  return cache_fwd_workspace_bytes(N, H, V);
}

int ikrl_lmhead_logprob_fwd_cached(const void* hidden, const void* weight, const int64_t* ids, int64_t N, int32_t H,
                                   int32_t V, float* logp, float* lse, const uint8_t* cache_mask, int64_t cache_rows,
                                   int32_t* cache_slot, void* cache_q, float* cache_m, void* ws, size_t ws_bytes,
                                   void* stream) {
  clear_error();
  const char* what = "ikrl_lmhead_logprob_fwd_cached";
  IKRL_REQUIRE(V % 8 == 0, IKRL_ERR_UNSUPPORTED, "%s: the logit cache needs V (%d) to be a multiple of 8", what, V);
  IKRL_REQUIRE(cache_rows >= 0, IKRL_ERR_INVALID_ARGUMENT, "%s: cache_rows %lld < 0", what, (long long)cache_rows);
  IKRL_REQUIRE(N == 0 || (cache_slot && lse && (cache_rows == 0 || (cache_q && cache_m))), IKRL_ERR_INVALID_ARGUMENT,
               "%s: null pointer", what);
  IKRL_REQUIRE((reinterpret_cast<uintptr_t>(cache_q) & 15) == 0 && (reinterpret_cast<uintptr_t>(cache_m) & 3) == 0,
               IKRL_ERR_ALIGNMENT, "%s: cache_q must be 16-byte and cache_m 4-byte aligned", what);
  const size_t need = N > 0 ? cache_fwd_workspace_bytes(N, H, V) : 0;
  IKRL_REQUIRE(N == 0 || (ws != nullptr && ws_bytes >= need), IKRL_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes",
               what, ws_bytes, need);
  CacheArgs c;
  c.mask = cache_mask;
  c.cap = cache_rows;
  c.slot = cache_slot;
  c.q = reinterpret_cast<uint16_t*>(cache_q);
  c.m = cache_m;
  return lmhead_fwd_impl(what, hidden, weight, ids, N, H, V, 0, false, logp, lse, ws, ws_bytes, stream, c);
}

int ikrl_lmhead_logprob_bwd_cached(const void* hidden, const void* weight, const int64_t* ids, const float* lse,
                                   const float* dlogp, int64_t N, int32_t H, int32_t V, int64_t chunk_rows,
                                   void* dhidden, void* dweight, int32_t dweight_dtype, int32_t accumulate_dweight,
                                   const int32_t* cache_slot, const void* cache_q, const float* cache_m, void* ws,
                                   size_t ws_bytes, void* stream) {
  clear_error();
  IKRL_REQUIRE(V % 8 == 0, IKRL_ERR_UNSUPPORTED, "ikrl_lmhead_logprob_bwd_cached: the logit cache needs V (%d) to "
               "be a multiple of 8", V);
  IKRL_REQUIRE(N == 0 || (cache_slot && cache_q && cache_m), IKRL_ERR_INVALID_ARGUMENT,
               "ikrl_lmhead_logprob_bwd_cached: null cache pointer");
  return lmhead_bwd_impl("ikrl_lmhead_logprob_bwd_cached", hidden, weight, ids, lse, dlogp, N, H, V, 0, chunk_rows,
                         dhidden, dweight, dweight_dtype, accumulate_dweight, ws, ws_bytes, stream, cache_slot,
                         reinterpret_cast<const uint16_t*>(cache_q), cache_m);
}

int ikrl_lmhead_shard_bwd(const void* hidden, const void* weight_shard, const int64_t* ids, const float* lse,
                          const float* dlogp, int64_t N, int32_t H, int32_t V_shard, int64_t vocab_start,
                          int64_t chunk_rows, void* dhidden_partial, void* dweight_shard, int32_t dweight_dtype,
                          int32_t accumulate_dweight, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  IKRL_REQUIRE(vocab_start >= 0, IKRL_ERR_INVALID_ARGUMENT, "ikrl_lmhead_shard_bwd: vocab_start %lld < 0",
               (long long)vocab_start);
  return lmhead_bwd_impl("ikrl_lmhead_shard_bwd", hidden, weight_shard, ids, lse, dlogp, N, H, V_shard, vocab_start,
                         chunk_rows, dhidden_partial, dweight_shard, dweight_dtype, accumulate_dweight, ws, ws_bytes,
                         stream);
}

int ikrl_lmhead_set_cta_pairs(int32_t enable) {
  int64_t prev = 1;
  ikrl_set_tuning(IKRL_TUNE_CTA_PAIRS, enable ? 1 : 0, &prev);
  return (int)prev;
}

int ikrl_lmhead_plan(int32_t gemm, int64_t rows, int32_t H, int32_t V, int32_t num_sms, int32_t* plan_out) {
  clear_error();
  IKRL_REQUIRE(gemm >= 0 && gemm <= 4, IKRL_ERR_INVALID_ARGUMENT, "ikrl_lmhead_plan: gemm %d not in 0..4", gemm);
  IKRL_REQUIRE(rows > 0 && rows <= (int64_t)65535 * BM && H > 0 && V > 0 && num_sms >= 2 && plan_out,
               IKRL_ERR_INVALID_ARGUMENT, "ikrl_lmhead_plan: bad arguments");
  const int64_t row_tiles = cdiv64(rows, BM);
  K1Plan pl{};
  if (gemm == 0)  // forward: the hint is the workspace's split count
    pl = plan_k1(EPI_LSE, row_tiles, V, H, fwd_layout(rows, H, V).splits, num_sms);
  else if (gemm == 1)  // dS recompute of one backward chunk of `rows` rows
    pl = plan_k1(EPI_DLOGITS, row_tiles, V, H, choose_splits(row_tiles, (int)cdiv64(V, BN), H), num_sms);
  else if (gemm == 2)  // dW += dS^T h over the chunk, fp32 accumulator
    pl = plan_k1(EPI_F32, cdiv64(V, BM), H, (int)rows, 0, num_sms);
  else if (gemm == 3)  // dH = dS W of the chunk, undivided
    pl = plan_k1(EPI_STORE_BF16, row_tiles, H, V, 0, num_sms);
  if (gemm == 4) {  // K ranges of that dH (1 = undivided), with the partial buffer of such a chunk
    const int64_t part = std::min<int64_t>(kSplitKPartElems, (int64_t)kMaxDhSplitK * rows * H);
    plan_out[0] = dh_split_k(row_tiles, H, V, rows, part, num_sms);
    plan_out[1] = plan_out[2] = plan_out[3] = 0;
    return IKRL_OK;
  }
  plan_out[0] = pl.kind;
  plan_out[1] = pl.n_tiles;
  plan_out[2] = pl.tiles_per_split;
  plan_out[3] = pl.splits;
  return IKRL_OK;
}

int ikrl_lmhead_status(const void* ws, int32_t* status_out, void* stream) {
  clear_error();
  IKRL_REQUIRE(ws && status_out, IKRL_ERR_INVALID_ARGUMENT, "ikrl_lmhead_status: null pointer");
  cudaStream_t s = as_stream(stream);
  int v = 0;
  IKRL_CUDA(cudaMemcpyAsync(&v, ws, sizeof(int), cudaMemcpyDeviceToHost, s));
  IKRL_CUDA(cudaStreamSynchronize(s));
  *status_out = v;
  if (v != 0) {
    set_error("device error 0x%x recorded by a tensor-core kernel (bounded wait expired)", v);
    return IKRL_ERR_DEVICE;
  }
  return IKRL_OK;
}

}  // extern "C"

// ---- allocation-free forward -------------------------------------------------------------------
//
// Some callers cannot allocate device memory at the moment they need log-probs: hosts that embed
// this library behind their own device-memory manager and forbid side allocations, frameworks
// that have already reserved all free memory in their caching pool (a cudaMalloc there fails or
// forces the pool to release memory and synchronise the device), and callers on a latency-critical
// path where an allocation's implicit synchronisation is not acceptable.  For them the forward
// below takes its scratch (the per-split row statistics and the device error word) from a fixed
// array compiled into the library instead of a caller-provided workspace.
//
// Limits and sharing rules:
//   * the array is kNoAllocScratchBytes (4 MiB) and lives on every GPU that loads the library
//     until the process exits; calls whose scratch would not fit are rejected with
//     IKRL_ERR_WORKSPACE (the message gives the sizes) -- use ikrl_lmhead_logprob_fwd instead;
//   * every call on a device uses the same array: calls whose kernels may overlap on the GPU
//     (different streams without ordering) race on it, so order them on one stream;
//   * the array keeps whatever the last call left in it; the error word at its start is cleared
//     by every call, the rest is fully rewritten before it is read;
//   * a bounded wait that expires inside a tensor-core kernel records a code in that error word
//     and the outputs become NaN; ikrl_lmhead_noalloc_status reads the word of the current device;
//   * the first call on each device looks up the device addresses of the library's two static
//     arrays (this scratch and the pacing counters of the wide kernel) with cudaGetSymbolAddress,
//     with that device current; make that first call before any stream capture begins.

namespace ikrl {
namespace {

constexpr size_t kNoAllocScratchBytes = size_t(4) << 20;
static __device__ __align__(256) unsigned char g_noalloc_scratch[kNoAllocScratchBytes];

constexpr int kMaxDevices = 64;
std::mutex g_noalloc_mu;
void* g_noalloc_addr[kMaxDevices] = {nullptr};

// Device address of g_noalloc_scratch on the current device, looked up once per device.  The
// same first call also resolves the pacing array, so that no later call on this device needs a
// symbol lookup, whatever its sizes.
int noalloc_scratch(void** out) {
  int dev = 0;
  IKRL_CUDA(cudaGetDevice(&dev));
  IKRL_REQUIRE(dev >= 0 && dev < kMaxDevices, IKRL_ERR_UNSUPPORTED, "device ordinal %d out of range", dev);
  std::lock_guard<std::mutex> lock(g_noalloc_mu);
  if (g_noalloc_addr[dev] == nullptr) {
    unsigned* pace = nullptr;
    int rc = pace_array(&pace);
    if (rc) return rc;
    void* p = nullptr;
    IKRL_CUDA(cudaGetSymbolAddress(&p, g_noalloc_scratch));
    g_noalloc_addr[dev] = p;
  }
  *out = g_noalloc_addr[dev];
  return IKRL_OK;
}

}  // namespace
}  // namespace ikrl

extern "C" int ikrl_lmhead_logprob_fwd_noalloc(const void* hidden, const void* weight, const int64_t* ids,
                                               int64_t N, int32_t H, int32_t V, float* logp, float* lse,
                                               void* stream) {
  clear_error();
  int rc = check_common(hidden, weight, ids, N, H, V, "ikrl_lmhead_logprob_fwd_noalloc");
  if (rc) return rc;
  const size_t need = ikrl_lmhead_fwd_workspace_bytes(N, H, V);
  IKRL_REQUIRE(need <= kNoAllocScratchBytes, IKRL_ERR_WORKSPACE,
               "ikrl_lmhead_logprob_fwd_noalloc: N=%lld rows (H=%d, V=%d) need %zu bytes of scratch, more than the "
               "built-in %zu; split the rows or call ikrl_lmhead_logprob_fwd with a workspace",
               (long long)N, H, V, need, kNoAllocScratchBytes);
  void* scratch = nullptr;
  if ((rc = noalloc_scratch(&scratch))) return rc;
  return ikrl_lmhead_logprob_fwd(hidden, weight, ids, N, H, V, logp, lse, scratch, kNoAllocScratchBytes, stream);
}

extern "C" int ikrl_lmhead_noalloc_status(int32_t* status_out, void* stream) {
  clear_error();
  IKRL_REQUIRE(status_out != nullptr, IKRL_ERR_INVALID_ARGUMENT, "ikrl_lmhead_noalloc_status: null pointer");
  void* scratch = nullptr;
  int rc = noalloc_scratch(&scratch);
  if (rc) return rc;
  return ikrl_lmhead_status(scratch, status_out, stream);
}
