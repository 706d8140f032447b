// Reading a row of logits (bf16 or fp32, any alignment) eight columns at a time, and the running
// (maximum, sum of 2^(c x - c maximum)) of what was read.
#pragma once

#include "common.cuh"

namespace ikrl {

// Columns [8 j - shift, 8 j - shift + 8) form group j: groups start on 16-byte boundaries whatever
// the row's own alignment, so every group but the first and the last of a row is loaded with
// 16-byte loads.
template <typename T>
struct RowView {
  const T* row;
  int V, shift, groups;
  __device__ __forceinline__ RowView(const T* base, int64_t ld, int64_t r, int V_) : row(base + r * ld), V(V_) {
    shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    groups = (V + shift + 7) >> 3;
  }
  __device__ __forceinline__ int first(int j) const { return 8 * j - shift; }
  __device__ __forceinline__ bool whole(int j) const { return first(j) >= 0 && first(j) + 8 <= V; }
};

// One part of a row of logits: part `seg` of `segs`, in groups of eight columns.
template <typename T>
struct RowPart {
  RowView<T> rv;
  int j0, j1;  // its groups
  int a, b;    // those of them that lie wholly inside the row
  __device__ __forceinline__ RowPart(const T* base, int64_t ld, int64_t r, int V, int seg, int segs)
      : rv(base, ld, r, V) {
    const int per = (rv.groups + segs - 1) / segs;
    j0 = min(seg * per, rv.groups);
    j1 = min(j0 + per, rv.groups);
    a = max(j0, rv.shift > 0 ? 1 : 0);
    b = max(a, min(j1, (V + rv.shift) >> 3));
  }
  __device__ __forceinline__ int group_of(int col) const { return (col + rv.shift) >> 3; }
  __device__ __forceinline__ const T* at(int j) const { return rv.row + rv.first(j); }
  // Edge t (0, 1): the group at the front or the back of the part that reaches past the row, or -1.
  __device__ __forceinline__ int edge(int t) const {
    return (t == 0 && a > j0) ? j0 : (t == 1 && b < j1 && j1 - 1 >= a) ? j1 - 1 : -1;
  }
};

// Two fp32 values in one 64-bit register, and the instructions that work on both at once.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
// 2^v of both.
__device__ __forceinline__ uint64_t exp2x2(uint64_t v) {
  float lo, hi;
  unpack2(v, lo, hi);
  return pack2(fast_exp2(lo), fast_exp2(hi));
}

template <typename T>
struct Group8;
template <>
struct Group8<uint16_t> {
  uint32_t w[4];
  __device__ __forceinline__ float get(int k) const { return (k & 1) ? bf16hi(w[k >> 1]) : bf16lo(w[k >> 1]); }
  __device__ __forceinline__ uint64_t get2(int k) const { return pack2(bf16lo(w[k]), bf16hi(w[k])); }
  // The largest value, NaN aside (-inf when there is no other).
  __device__ __forceinline__ float max() const {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(fmaxf(__low2float(m), __high2float(m)), -INFINITY);
  }
  // Value `rel` of the group, which becomes -inf.
  __device__ __forceinline__ float take(int rel) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k == rel) {
        x = get(k);
        w[k >> 1] = (k & 1) ? ((w[k >> 1] & 0xffffu) | 0xff800000u) : ((w[k >> 1] & 0xffff0000u) | 0xff80u);
      }
    return x;
  }
  __device__ __forceinline__ void load(const uint16_t* p);
  __device__ __forceinline__ void fill() { w[0] = w[1] = w[2] = w[3] = 0xff80ff80u; }
};
template <>
struct Group8<float> {
  uint32_t w[8];
  __device__ __forceinline__ float get(int k) const { return __uint_as_float(w[k]); }
  __device__ __forceinline__ uint64_t get2(int k) const { return pack2(get(2 * k), get(2 * k + 1)); }
  __device__ __forceinline__ float max() const {
    return fmaxf(fmaxf(fmaxf(fmaxf(get(0), get(1)), fmaxf(get(2), get(3))),
                       fmaxf(fmaxf(get(4), get(5)), fmaxf(get(6), get(7)))), -INFINITY);
  }
  __device__ __forceinline__ float take(int rel) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k == rel) {
        x = get(k);
        w[k] = 0xff800000u;
      }
    return x;
  }
  __device__ __forceinline__ void load(const float* p);
  __device__ __forceinline__ void fill() {
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = 0xff800000u;
  }
};

__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void st_stream16(void* p, uint4 v) {
  asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

__device__ __forceinline__ void Group8<uint16_t>::load(const uint16_t* p) {
  const uint4 v = ld_stream16(p);
  w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
}
__device__ __forceinline__ void Group8<float>::load(const float* p) {
  const uint4 v = ld_stream16(p), u = ld_stream16(p + 4);
  w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  w[4] = u.x; w[5] = u.y; w[6] = u.z; w[7] = u.w;
}

// Group j of the row; columns outside the row read as -inf.
template <typename T>
__device__ __forceinline__ void load_group(Group8<T>& g, const RowView<T>& rv, int j) {
  const int v0 = rv.first(j);
  if (rv.whole(j)) {
    g.load(rv.row + v0);
    return;
  }
  g.fill();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int a = v0 + k;
    if (a < 0 || a >= rv.V) continue;
    if constexpr (sizeof(T) == 2) {
      const uint32_t b = rv.row[a];
      g.w[k >> 1] = (k & 1) ? ((g.w[k >> 1] & 0xffffu) | (b << 16)) : ((g.w[k >> 1] & 0xffff0000u) | b);
    } else {
      g.w[k] = __float_as_uint(rv.row[a]);
    }
  }
}

// Below this size of c m its rounding is at most half of one log2 unit, and exponents are formed with one
// fma from the rounded value.  (At -1e30, a common mask, the rounding alone would be 10^22 units.)
constexpr float kFmaLimit = 1e7f;

// Running (m, s) over U more groups: m the maximum, s the sum of 2^(c (x - m)).  One maximum and one
// rescaling serve all of them; then two values cost two unpackings, a packed fma, two exponentials and
// a packed addition.  The fma takes c x from the rounded c m, and what that rounding leaves is
// multiplied out once per call, so the sum stands relative to m itself.
//
// A mask may hold -1e30 or the type's lowest value: there the difference x - m is taken first.  While nothing but
// -inf was seen the sum is taken from 0, which leaves it 0; NaN and +inf make it NaN.
// top[u]: the groups' own maxima, NaN aside.  done(u) is called when g[u] is used up.
template <typename T, int U, typename Done>
__device__ __forceinline__ void online_groups(Group8<T> (&g)[U], float c, float& m, float& s, float (&top)[U],
                                              Done done) {
#pragma unroll
  for (int u = 0; u < U; ++u) top[u] = g[u].max();
  float mx = top[0];
#pragma unroll
  for (int u = 1; u < U; ++u) mx = fmaxf(mx, top[u]);
  if (mx > m) {
    s *= fast_exp2((m - mx) * c);
    m = mx;
  }
  const float pt = m * c;
  if (fabsf(pt) < kFmaLimit) {
    const uint64_t c2 = pack2(c, c), npt2 = pack2(-pt, -pt);
    uint64_t b0 = 0, b1 = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        b0 = add2(b0, exp2x2(fma2(g[u].get2(k), c2, npt2)));
        b1 = add2(b1, exp2x2(fma2(g[u].get2(k + 1), c2, npt2)));
      }
      done(u);
    }
    float lo, hi;
    unpack2(add2(b0, b1), lo, hi);
    s = fmaf(lo + hi, fast_exp2(-fmaf(m, c, -pt)), s);
  } else {
    const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < 8; ++k) s += fast_exp2((g[u].get(k) - from) * c);
      done(u);
    }
  }
}

template <typename T, int U>
__device__ __forceinline__ void online_groups(Group8<T> (&g)[U], float c, float& m, float& s) {
  float top[U];
  online_groups<T, U>(g, c, m, s, top, [](int) {});
}

__device__ __forceinline__ void online_merge(float c, float& m, float& s, float m2, float s2) {
  const float mm = fmaxf(m, m2);
  if (mm == -INFINITY) {
    s += s2;  // 0, or NaN that stays
    return;
  }
  s = s * fast_exp2((m - mm) * c) + s2 * fast_exp2((m2 - mm) * c);
  m = mm;
}

// Merge over the block, in a fixed order; every thread gets the result.  scratch: 64 floats.
__device__ __forceinline__ void block_online_merge(float c, float& m, float& s, float* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    online_merge(c, m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if (lane == 0) {
    scratch[warp] = m;
    scratch[32 + warp] = s;
  }
  __syncthreads();
  m = lane < nw ? scratch[lane] : -INFINITY;
  s = lane < nw ? scratch[32 + lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    online_merge(c, m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
}

// Blocks (of one cluster) that share a row: the power of two up to 8 with which all blocks still run at
// once, two an SM, and each keeps a column range of `min_groups` groups.  (Top 64 of 64 rows of 151936 bf16
// columns: 25 us in clusters of 4, 41 us in clusters of 8; of 100 rows 27 us in 2, 37 us in 4.)
inline int row_cluster(int64_t N, int V, int min_groups) {
  int c = 1;
  while (c < 8 && 2 * N * c <= 2 * kNumSMs && V / 8 / (2 * c) >= min_groups) c *= 2;
  return c;
}

// How many rows are read by one block each, and into how many parts the others are cut.  An SM holds four blocks
// and reads 44 bytes a ns (of 6.5 TB/s), and each of its rounds of four costs about 2.8 us beside the bytes
// (forward of 4096 rows of 151936 bf16 columns in 1, 2, 4, 8 parts: 237, 257, 329, 479 us), so rows are cut only
// where the SMs would not come out even otherwise and 5% is to be had: all of them, or those that are left when
// every SM has as many whole rows.  A part keeps at least `round` groups.  (Forward of 300 / 512 such
// rows: 45 / 53 us, 48 / 56 with all rows cut alike; 512 rows of 50257 columns: 35 us against 38.)
constexpr int kMaxRowParts = 8;
struct RowCut {
  int64_t whole;  // rows [0, whole) are whole
  int parts;      // parts of each of the others
};
inline RowCut row_cut(int64_t N, int V, int elem_bytes, int round) {
  const double row_us = (double)V * elem_bytes / 44e3;
  RowCut best{0, 1};
  double least = 0.0;
  for (int q = 1; q <= kMaxRowParts && (q == 1 || V / 8 / q >= round); q *= 2) {
    for (const int64_t whole : {(int64_t)0, N / kNumSMs * kNumSMs}) {
      const int64_t parts = (N - whole) * q;
      const double rows = (double)(whole / kNumSMs) + (double)((parts + kNumSMs - 1) / kNumSMs) / q;
      const double us = rows * row_us + (double)((whole + parts + 4 * kNumSMs - 1) / (4 * kNumSMs)) * 2.8;
      if (least == 0.0 || us < 0.95 * least) {
        least = us;
        best = {whole, q};
      }
    }
  }
  return best;
}

}  // namespace ikrl
