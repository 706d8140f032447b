// Losses between a row's softmax and a few named outcomes: distillation from a teacher's top
// log-probs and cross entropy.  Shared by the kernels that read logits (distill.cu) and by the LM
// head (lmhead.cu).
//
// A row has logits x_v, z = x / T, p = softmax(z), and up to K named columns ("entries"): the
// teacher's tokens with log-probs l_k, q_k = exp(l_k), or the one target of a cross entropy.  The
// other columns are the tail.  Every loss here depends on p through the entries' p_k and the tail's
// total p_t only, so its gradient is
//     dL/dx_k = grad_k                      at the entries,
//     dL/dx_v = coef * softmax_tail(x)_v    at the others   (plus a constant for label smoothing),
// with softmax_tail normalised over the tail alone and coef = p_t * (dL/dp_t - sum_j p_j dL/dp_j) / T.
// The tail's sum is formed from the tail's own columns (never 1 - sum p_k, which cancels when the
// student is sure), and no quotient by p_t appears, so rows with a vanishing tail stay finite.
#pragma once

#include "common.cuh"

namespace ikrl {

constexpr int kMaxEntries = 256;           // entries a row may have
constexpr int kMaxVocab = 1 << 21;         // columns of the kernels on logits
constexpr int kMaxParts = 8;               // parts a row of logits may be cut into
constexpr int kNoEntry = 0x7fffffff;       // pads a row's sorted entry columns
constexpr double kTailEps = 1.0 / (1 << 20);
// Sums of logits in memory are kept in this unit, a power of two above their number: a row masked with the
// type's lowest value has a mean in range although its plain sum is not.
constexpr float kSumUnit = 4194304.f;
static_assert(kMaxVocab < 4194304, "the unit keeps every row's sum in range");

// What a row's id says (the compaction of the LM-head backward skips kRowNone rows).
constexpr int64_t kRowNone = -100;  // no entries (or an ignored target): loss 0, no gradient
constexpr int64_t kRowLive = -1;
constexpr int64_t kRowBad = -2;     // names a column outside the vocabulary: NaN

enum RowLoss : int {
  ROW_FORWARD = 0,       // KL(q | p), tail as one more outcome
  ROW_FORWARD_TOPK = 1,  // KL(q / sum q | p), no tail outcome
  ROW_REVERSE = 2,       // KL(p | q)
  ROW_JSD = 3,           // b KL(q | m) + (1 - b) KL(p | m), m = b q + (1 - b) p
  ROW_XENT = 4           // cross entropy with label smoothing and a z term
};

struct RowLossParams {
  int loss;
  int V;
  float c;      // log2(e) / T: logits to log2 units
  float inv_t;  // 1 / T
  float beta;   // ROW_JSD
  float smoothing, zeta;  // ROW_XENT
  float sum_unit;         // ROW_XENT: unit of the sums of all logits
};

// What a forward keeps for its backward, in one caller-owned buffer.
struct RowState {
  int64_t* row_ids;  // [N] kRowNone / kRowLive / kRowBad
  float* ref;        // [N] logit the tail is normalised from: softmax_tail = 2^(c (x - ref)), up to
                     //     a factor that coef holds
  float* coef;       // [N]
  int* cols;         // [N][K] entry columns ascending, then kNoEntry
  float* grad;       // [N][K] gradient at them (until the loss is formed: the teacher's log-probs)
  float* xk;         // [N][K] logits at them (forward only)
  float* part;       // [3][kMaxParts][N] tail maxima and sums, sums of all logits, per part of a row
                     //     (forward on logits only)
};

inline size_t row_state_bytes(int64_t N, int K) {
  auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
  return al((size_t)N * 8) + 2 * al((size_t)N * 4) + 3 * al((size_t)N * K * 4) +
         al((size_t)N * 12 * kMaxParts);
}

inline RowState row_state(void* base, int64_t N, int K) {
  auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
  char* p = reinterpret_cast<char*>(base);
  RowState s;
  s.row_ids = reinterpret_cast<int64_t*>(p); p += al((size_t)N * 8);
  s.ref = reinterpret_cast<float*>(p); p += al((size_t)N * 4);
  s.coef = reinterpret_cast<float*>(p); p += al((size_t)N * 4);
  s.cols = reinterpret_cast<int*>(p); p += al((size_t)N * K * 4);
  s.grad = reinterpret_cast<float*>(p); p += al((size_t)N * K * 4);
  s.xk = reinterpret_cast<float*>(p); p += al((size_t)N * K * 4);
  s.part = reinterpret_cast<float*>(p);
  return s;
}

// Checks of the C entries (distill.cu): sizes, types and alignment of logits in memory; the
// parameters of a loss, turned into RowLossParams.
int check_logits_arg(const char* what, const void* logits, int32_t dtype, int64_t ld, int64_t N, int32_t V);
int distill_params(const char* what, const ikrl_distill_params* d, int V, int K, RowLossParams* out);
int xent_params(const char* what, float smoothing, float z_loss, int V, RowLossParams* out);

// Few rows come with many partial sets (a GEMM of one row tile cuts the columns as fine as it can): a block a row
// joins them, otherwise a warp.
inline bool row_takes_a_block(int sets, int64_t N) { return sets > 64 && N <= 4 * kNumSMs; }

// The LM head's use of the two kernels in distill.cu: entries before its GEMM, losses after it.
// tids / tlp: the teacher's [N][K], or targets with K = 1 and tlp null (ROW_XENT); clear: a word to
// zero, or null.
int launch_row_entries(const int64_t* tids, const float* tlp, int64_t N, int K, const RowLossParams& p,
                       const RowState& st, cudaStream_t s, int* clear = nullptr);
// part_m / part_s / part_x: [sets][N] tail maxima, sums of 2^(c (x - max)), plain sums of all logits
// (part_x null without label smoothing), the number of sets on the device where sets_dev is given; pos: the
// place of each row in them, or null: itself; err: an error word that makes every loss NaN, or null.
int launch_row_losses(const float* part_m, const float* part_s, const float* part_x, int sets, const int* sets_dev,
                      const int* pos, int64_t N, int K, const RowLossParams& p, const RowState& st, float* loss,
                      const int* err, cudaStream_t s);

// ---- device side ---------------------------------------------------------------------------------

__device__ __forceinline__ float nan_f32() { return __int_as_float(0x7fc00000); }

// Threads that order a row's K entries.
__host__ __device__ inline int entry_threads(int K) {
  int n = 32;
  while (n < K) n *= 2;
  return n;
}

// One row's entries, by a block of at least entry_threads(K) threads: columns ascending into s_col
// (kNoEntry behind the last) and the teacher's log-probs beside them into s_lp.  An entry counts
// when its id is >= 0 and its log-prob is not -inf, and a repeated id at its first place only.
// s_raw: kMaxEntries scratch words.  Returns the row's id; cnt = entries that count.
// A bitonic sort of (column, place), one a thread (256 entries of 4096 rows: 30 us; 83 us when every
// entry counted the smaller ones).
__device__ __forceinline__ int64_t row_entries(const int64_t* __restrict__ tids, const float* __restrict__ tlp, int K,
                                               int V, int* s_col, float* s_lp, int* s_raw, int& cnt) {
  if (tlp == nullptr) {  // one target
    const int64_t t = tids[0];
    const bool ok = t >= 0 && t < V;
    if (threadIdx.x == 0) {
      s_col[0] = ok ? (int)t : kNoEntry;
      s_lp[0] = 0.f;
    }
    __syncthreads();
    cnt = ok ? 1 : 0;
    return ok ? kRowLive : (t == -100 ? kRowNone : kRowBad);
  }
  const int t = threadIdx.x, n = entry_threads(K);
  constexpr uint32_t kNone = 0xffffffffu;
  uint32_t key = kNone;
  bool bad = false;
  if (t < K) {
    const int64_t id = tids[t];
    const bool use = id >= 0 && !(tlp[t] == -INFINITY);  // a NaN log-prob counts (row_loss makes the row NaN)
    bad = use && id >= V;
    if (use && !bad) key = (uint32_t)id << 8 | (uint32_t)t;
  }
  const bool any_bad = __syncthreads_or(bad);
  uint32_t* word = reinterpret_cast<uint32_t*>(s_raw);
  for (int k = 2; k <= n; k <<= 1) {
    const bool up = (t & k) == 0;
    for (int j = k >> 1; j > 0; j >>= 1) {
      uint32_t other;
      if (j >= 32) {
        __syncthreads();
        if (t < n) word[t] = key;
        __syncthreads();
        other = t < n ? word[t ^ j] : key;
      } else {
        other = __shfl_xor_sync(0xffffffffu, key, j);
      }
      key = ((t & j) == 0) == up ? min(key, other) : max(key, other);
    }
  }
  __syncthreads();
  if (t < n) word[t] = key;
  __syncthreads();
  const bool repeat = t > 0 && t < n && key != kNone && word[t - 1] >> 8 == key >> 8;
  const bool keep = t < n && key != kNone && !repeat;
  int rank = t;
  if (__syncthreads_or(repeat)) {  // those behind a repeat move up
    const uint32_t kept = __ballot_sync(0xffffffffu, keep);
    if ((t & 31) == 0 && t < n) word[t >> 5] = __popc(kept);
    __syncthreads();
    rank = __popc(kept & ((1u << (t & 31)) - 1u));
    for (int w = 0; w < (t >> 5) && t < n; ++w) rank += (int)word[w];
  }
  cnt = __syncthreads_count(keep);
  if (keep) {
    s_col[rank] = (int)(key >> 8);
    s_lp[rank] = tlp[key & 255u];
  }
  if (t >= cnt && t < K) {
    s_col[t] = kNoEntry;
    s_lp[t] = 0.f;
  }
  __syncthreads();
  return any_bad ? kRowBad : (cnt == 0 ? kRowNone : kRowLive);
}

// One row's loss and gradient by one warp.  x[k], lp[k], k < cnt: the logits and teacher log-probs
// of its entries; the tail has maximum tm and sum ts of 2^(c (x - tm)); sum_x: the sum of all logits in
// units of P.sum_unit (ROW_XENT).  Writes *loss, *ref, *coef and grad[k] (grad may be lp's array: each lane reads its
// entries before it writes them).
//
// log p is formed as (x - m) / T - log(s) with the row's maximum m: both terms are small, so nothing
// of an entry's log-prob is lost to the size of the logits, and a mask of the type's lowest value
// stays finite.
__device__ inline void row_loss(const RowLossParams& P, int64_t row_id, int cnt, const float* x, const float* lp,
                                float tm, float ts, float sum_x, float* loss, float* ref, float* coef, float* grad) {
  const int lane = threadIdx.x & 31;
  if (row_id != kRowLive) {
    const float v = row_id == kRowNone ? 0.f : nan_f32();
    for (int k = lane; k < cnt; k += 32) grad[k] = v;
    if (lane == 0) {
      *loss = v;
      *ref = INFINITY;
      *coef = v;
    }
    return;
  }
  const bool rest = ts != 0.f;  // some tail column is above -inf (NaN counts, and stays)
  float m = rest ? tm : -INFINITY;
  for (int k = lane; k < cnt; k += 32) m = fmaxf(m, x[k]);
  m = warp_max(m);
  float s = 0.f;
  for (int k = lane; k < cnt; k += 32) s += exp2f((x[k] - m) * P.c);
  s = warp_sum(s);
  const float tail_s = rest ? ts * exp2f((tm - m) * P.c) : 0.f;
  s += tail_s;
  const float ls = log2f(s);
  const float log_pt = rest ? (tm - m) * P.inv_t + (log2f(ts) - ls) * kLn2 : -INFINITY;
  const float pt = tail_s / s;
  // ref is the tail's log-sum as a logit, rounded; what the rounding leaves goes into coef.
  float r = INFINITY, fix = 0.f;
  if (rest) {
    r = tm + log2f(ts) / P.c;
    fix = exp2f((r - tm) * P.c - log2f(ts));
  }

  if (P.loss == ROW_XENT) {
    if (lane == 0) {
      const float xy = x[0];
      const float lse = m + ls * kLn2;
      // -log p of the target: log1p of the others' sum over its own where that is the smaller
      const float nll = (rest && tm > xy) ? ls * kLn2 - (xy - m)
                                          : log1pf(rest ? ts * exp2f((tm - xy) * P.c) : 0.f);
      const float mean = P.smoothing != 0.f ? sum_x / (float)P.V * P.sum_unit : 0.f;
      const float smooth = P.smoothing != 0.f ? P.smoothing * (xy - mean) : 0.f;
      *loss = nll + smooth + P.zeta * lse * lse;
      const float a1 = 2.f * P.zeta * lse;
      const float py = exp2f((xy - m) * P.c) / s;
      *ref = r;
      *coef = (1.f + a1) * pt * fix;
      grad[0] = a1 * py - pt + P.smoothing * (1.f - 1.f / (float)P.V);
    }
    return;
  }

  // The teacher's mass in 64 bits: 1 - Q is what the tail outcome gets.
  double q64 = 0.0;
  for (int k = lane; k < cnt; k += 32) q64 += exp((double)lp[k]);
  q64 = warp_sum(q64);
  if (q64 != q64) {  // an entry's log-prob is NaN: so are the row's loss and gradient
    for (int k = lane; k < cnt; k += 32) grad[k] = nan_f32();
    if (lane == 0) {
      *loss = nan_f32();
      *ref = r;
      *coef = nan_f32();
    }
    return;
  }
  // ROW_FORWARD_TOPK renormalises the teacher over its entries: log q = lp - top - lq64.  Where their mass leaves
  // the range of 64 bits (entries near e^-745 and below) it is summed from its largest.
  double top = 0.0, lq64 = 0.0;
  if (P.loss == ROW_FORWARD_TOPK) {
    double mass = q64;
    if (q64 < 1e-290) {
      float hi = -INFINITY;
      for (int k = lane; k < cnt; k += 32) hi = fmaxf(hi, lp[k]);
      top = (double)warp_max(hi);
      mass = 0.0;
      for (int k = lane; k < cnt; k += 32) mass += exp((double)lp[k] - top);
      mass = warp_sum(mass);
    }
    lq64 = log(mass);
  }
  const double left = 1.0 - q64;
  const bool columns_left = cnt < P.V;
  float qt = 0.f, log_qt = 0.f;
  if (P.loss != ROW_FORWARD_TOPK && columns_left) {
    qt = left >= kTailEps ? (float)left : 0.f;
    log_qt = (float)log(left >= kTailEps ? left : kTailEps);
  }
  const float b = P.beta, log_b = logf(b), log_1b = log1pf(-b);
  float sum = 0.f, mean = 0.f;  // the loss, and sum_j p_j c_j
  // c_k and the entry's share of the loss; log_p, p: the student's, lq, q: the teacher's
  auto outcome = [&](float log_p, float p, float lq, float q, float& ck) -> float {
    if (P.loss == ROW_FORWARD || P.loss == ROW_FORWARD_TOPK) {
      ck = 0.f;
      return q > 0.f ? q * (lq - log_p) : 0.f;
    }
    if (P.loss == ROW_REVERSE) {
      ck = log_p - lq;
      return p > 0.f ? p * ck : (p == 0.f ? 0.f : p);
    }
    const float u = q > 0.f ? log_b + lq : -INFINITY, w = log_1b + log_p;
    const float hi = fmaxf(u, w);
    const float log_m = hi + log1pf(expf(fminf(u, w) - hi));
    ck = (1.f - b) * (log_p - log_m);
    const float first = q > 0.f ? b * q * (lq - log_m) : 0.f;
    return first + (p > 0.f ? p * ck : (p == 0.f ? 0.f : p));
  };
  for (int k = lane; k < cnt; k += 32) {
    const float log_p = (x[k] - m) * P.inv_t - ls * kLn2, p = exp2f((x[k] - m) * P.c - ls);
    const float lq = (float)((double)lp[k] - top - lq64);
    float ck;
    sum += outcome(log_p, p, lq, expf(lq), ck);
    mean += p > 0.f ? p * ck : 0.f;
  }
  sum = warp_sum(sum);
  mean = warp_sum(mean);
  float ct = 0.f;
  if (P.loss != ROW_FORWARD_TOPK && columns_left) {
    sum += outcome(log_pt, pt, log_qt, qt, ct);
    mean += pt > 0.f ? pt * ct : 0.f;
  }
  const float S = P.loss == ROW_FORWARD_TOPK ? 1.f : (float)(q64 + (double)qt);
  for (int k = lane; k < cnt; k += 32) {
    const float log_p = (x[k] - m) * P.inv_t - ls * kLn2, p = exp2f((x[k] - m) * P.c - ls);
    const float lq = (float)((double)lp[k] - top - lq64);
    const float q = expf(lq);
    float d;
    if (P.loss == ROW_FORWARD || P.loss == ROW_FORWARD_TOPK) {
      d = S * p - q;
    } else {
      float ck;
      outcome(log_p, p, lq, q, ck);
      d = p > 0.f ? p * (ck - mean) : (p == 0.f ? 0.f : p);
    }
    grad[k] = d * P.inv_t;
  }
  if (lane == 0) {
    float a;
    if (P.loss == ROW_FORWARD) a = S * pt - qt;
    else if (P.loss == ROW_FORWARD_TOPK) a = pt;
    else a = pt > 0.f ? pt * (ct - mean) : (pt == 0.f ? 0.f : pt);
    *loss = sum;
    *ref = r;
    *coef = a * P.inv_t * fix;
  }
}

}  // namespace ikrl
