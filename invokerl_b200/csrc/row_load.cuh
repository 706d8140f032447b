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

template <typename T>
struct Group8;
template <>
struct Group8<uint16_t> {
  uint4 v;
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = bf16lo(w[k]);
      x[2 * k + 1] = bf16hi(w[k]);
    }
  }
};
template <>
struct Group8<float> {
  uint4 v, u;
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[8] = {v.x, v.y, v.z, v.w, u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(w[k]);
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

// Group j of the row; columns outside the row read as -inf.
__device__ __forceinline__ Group8<uint16_t> load_group(const RowView<uint16_t>& rv, int j) {
  Group8<uint16_t> g;
  const int v0 = rv.first(j);
  if (rv.whole(j)) {
    g.v = ld_stream16(rv.row + v0);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int a = v0 + 2 * k, b = a + 1;
      const uint32_t lo = (a >= 0 && a < rv.V) ? rv.row[a] : 0xff80u;
      const uint32_t hi = (b >= 0 && b < rv.V) ? rv.row[b] : 0xff80u;
      w[k] = lo | (hi << 16);
    }
    g.v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return g;
}
__device__ __forceinline__ Group8<float> load_group(const RowView<float>& rv, int j) {
  Group8<float> g;
  const int v0 = rv.first(j);
  if (rv.whole(j)) {
    g.v = ld_stream16(rv.row + v0);
    g.u = ld_stream16(rv.row + v0 + 4);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int a = v0 + k;
      w[k] = (a >= 0 && a < rv.V) ? __float_as_uint(rv.row[a]) : 0xff800000u;
    }
    g.v = make_uint4(w[0], w[1], w[2], w[3]);
    g.u = make_uint4(w[4], w[5], w[6], w[7]);
  }
  return g;
}

// Running (m, s) over eight more values: m the maximum, s the sum of 2^(c (x - m)).  The difference
// is taken before the product: c x may pass the range of fp32 where a mask holds the type's lowest
// value, x - m does not.  While nothing but -inf was seen the sum is taken from 0, which leaves it
// 0; NaN and +inf make it NaN.
__device__ __forceinline__ void online_update(const float (&x)[8], float c, float& m, float& s) {
  const float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  if (mx > m) {
    s *= fast_exp2((m - mx) * c);
    m = mx;
  }
  const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int k = 0; k < 8; ++k) s += fast_exp2((x[k] - from) * c);
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

// Blocks (of one cluster) that share a row: 1 when there are rows enough for every SM to hold two
// blocks, else the power of two up to 8 that gets there while each block keeps a column range of
// `min_groups` groups.
inline int row_cluster(int64_t N, int V, int min_groups) {
  int c = 1;
  while (c < 8 && N * c < 2 * kNumSMs && V / 8 / (2 * c) >= min_groups) c *= 2;
  return c;
}

}  // namespace ikrl
