// What the attention kernels over rows of a projection share (tree.hip, page_attend.hip): rows of f32 or f16 values as
// they stand, queries and softmax weights as the matrix cores take them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "xlane.h"

namespace rows {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
// The same loaded from and stored to 4-byte aligned places (one wide access all the same).
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x2 u32x2_a4 __attribute__((aligned(4)));
typedef floatx4 floatx4_a4 __attribute__((aligned(4)));

// How far scores may pass a row's maximum, in binary digits, before it is moved.
constexpr float SLACK = 4.0f;
// Exponents are taken as score * factor + (10 − maximum * factor), whose sum in brackets is rounded like a score; past
// this it would be off by whole digits, and the maximum is subtracted first.
constexpr float FAR = 65536.0f;
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16;
}
// Four values of a row as they stand, and as f16 pairs.
template <typename T>
struct Four {
  typedef floatx4 type;
};
template <>
struct Four<_Float16> {
  typedef u32x2 type;
};
__device__ __forceinline__ floatx4 raw4(const float *p) { return *(const floatx4_a4 *)p; }
__device__ __forceinline__ u32x2 raw4(const _Float16 *p) { return *(const u32x2_a4 *)p; }
__device__ __forceinline__ u32x2 pairs4(floatx4 x) { return u32x2{pack2(x[0], x[1]), pack2(x[2], x[3])}; }
__device__ __forceinline__ u32x2 pairs4(u32x2 x) { return x; }
template <typename T>
__device__ __forceinline__ u32x2 four(const T *p) { return pairs4(raw4(p)); }
// And in f32.
__device__ __forceinline__ void values(const float *p, float *f) { *(floatx4 *)f = raw4(p); }
__device__ __forceinline__ void values(const _Float16 *p, float *f) {
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  const half4 h = __builtin_bit_cast(half4, raw4(p));
#pragma unroll
  for (int e = 0; e < 4; e++) f[e] = (float)h[e];
}

// A pair of f16 values with zeros for those that are no finite numbers.
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  return ((w & 0x7c00u) == 0x7c00u ? 0u : w & 0xffffu) | ((w & 0x7c000000u) == 0x7c000000u ? 0u : w & 0xffff0000u);
}
// Value d of a row as f16 if it is no finite number, or zero.
template <typename T>
__device__ __forceinline__ float not_finite(const T *p, int d, int hd) {
  const float x = d < hd ? (float)(_Float16)p[d] : 0.0f;
  return isfinite(x) ? 0.0f : x;
}

// A barrier for what is in LDS: loads from memory stay under way.
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

__device__ __forceinline__ floatx4 mfma(half8 a, half8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Softmax weights p0 and p1 as f16, and (unless P16) what that leaves of them.
template <bool P16>
__device__ __forceinline__ void weights2(float p0, float p1, half8 &h, half8 &l, int e) {
  const half2 w = __builtin_convertvector((floatx2{p0, p1}), half2);
  h[e] = w[0], h[e + 1] = w[1];
  if constexpr (!P16) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w);
    floatx2 r;  // p − w, a product and a sum with a half as it stands
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(r[0]) : "v"(u), "v"(p0));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r[1]) : "v"(u), "v"(p1));
    const half2 x = __builtin_convertvector(r, half2);
    l[e] = x[0], l[e + 1] = x[1];
  }
}

// Row (of a key head's: node row / group, query head row % group) and head offset without a division where the heads
// are not shared.
__device__ __forceinline__ int node_of(int row, int group) { return group == 1 ? row : row / group; }
__device__ __forceinline__ int head_of(int row, int group) { return group == 1 ? 0 : row % group; }

// A row's query as the matrix cores take it (lane 16g + i: row i's 8 values from 8g on of every chunk of 32): its values,
// and those times a power of two and in two parts for f32 (precision is said at attend_kernel), with the factor of its
// scores' exponents.
template <typename T, int C>
__device__ __forceinline__ void load_query(const T *src, int g, int hd, float (&f)[C][8]) {
#pragma unroll
  for (int c = 0; c < C; c++)
#pragma unroll
    for (int y = 0; y < 2; y++) {
      const int d = 32 * c + 8 * g + 4 * y;
      values(src + (d < hd ? d : 0), &f[c][4 * y]);
#pragma unroll
      for (int e = 0; e < 4; e++) f[c][4 * y + e] = d < hd ? f[c][4 * y + e] : 0.0f;
    }
}
template <int C, int QP>
__device__ __forceinline__ float split_query(const float (&f)[C][8], float scale, half8 (&q)[C][QP]) {
  int k = 0;
  if constexpr (QP == 2) {
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(f[c][e]));
    top = xlane::bit4(top, xlane::Max{});
    top = xlane::bit5(top, xlane::Max{});
    if (top > 0.0f && top < INFINITY) k = min(8 - __builtin_amdgcn_frexp_expf(top), 100);  // its largest value into [2^7, 2^8)
  }
#pragma unroll
  for (int c = 0; c < C; c++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float y = QP == 2 ? ldexpf(f[c][e], k) : f[c][e];
      q[c][0][e] = (_Float16)y;
      if constexpr (QP == 2) q[c][1][e] = (_Float16)(y - (float)q[c][0][e]);
    }
  return ldexpf(scale * 1.44269504088896341f, -k);
}

}  // namespace rows
