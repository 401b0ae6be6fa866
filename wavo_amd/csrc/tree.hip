// A decoder step over trees of drafted tokens (include/wavo_hip.h, wh_tree): attention of every node over
// its sequence's f16 cache and the nodes that it sees, and the path of the tree that is kept.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "internal.h"
#include "xlane.h"

namespace {

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

struct AttendArgs {
  const void *q, *k, *v;
  size_t stride;
  const uint32_t *kv;
  size_t kv_stride;
  void *o;
  const int32_t *n, *count;
  const uint32_t *mask;
  size_t mask_stride;
  int batch, rows, words, cols, heads, kv_heads, hd;
  float scale;
  int kw, splits, row_blocks, block, node_block;  // (positions per block of the cache and of the nodes)
  // splits > 1: unnormalized outputs [split][batch * rows][heads][hd] and (maximum, sum, factor of the maximum's
  // exponent, -) [split][batch * rows][heads] of the splits that are used.
  float *po, *pml;
};

// How far scores may pass a row's maximum, in binary digits, before it is moved.
constexpr float SLACK = 4.0f;
// Exponents are taken as score * factor + (10 − maximum * factor), whose sum in brackets is rounded like a score; past
// this it would be off by whole digits, and the maximum is subtracted first.
constexpr float FAR = 65536.0f;
constexpr int WAVES = 8;  // wavefronts of a workgroup, at most

constexpr int few_block(int hd) { return hd <= 64 ? 64 : 32; }   // positions of a block of attend_kernel
constexpr int NODES = 32;                                        // (of its nodes: this many)
constexpr int rows_block(int hd) { return hd <= 64 ? 64 : 32; }  // and of attend_rows_kernel

// The blocks of keys of a sequence (the cache's, then the nodes'), and how its `splits` workgroups share them:
// runs of `per` blocks, at least one for each wavefront, so that a short sequence uses fewer of them.
struct Share {
  int n, count, cached, blocks, per, used;
};
__device__ __forceinline__ Share share_of(const AttendArgs &a, int b) {
  Share s;
  s.n = min(max(a.n[b], 0), a.cols);
  s.count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows;
  s.cached = (s.n + a.block - 1) / a.block;
  s.blocks = s.cached + (a.mask && a.k ? (s.count + a.node_block - 1) / a.node_block : 0);
  s.per = s.blocks, s.used = 1;
  if (a.splits > 1) {
    s.per = max((s.blocks + a.splits - 1) / a.splits, a.kw);
    s.used = max((s.blocks + s.per - 1) / s.per, 1);
  }
  return s;
}

// Whether node i of sequence b sees anything at all.
__device__ bool sees_any(const AttendArgs &a, const Share &s, int b, int i) {
  if (s.n > 0) return true;
  if (!a.mask || !a.k) return false;
  const uint32_t *w = a.mask + (size_t)b * a.mask_stride + (size_t)i * a.words;
  for (int j = 0; j < s.count; j += 32)
    if (w[j / 32] & (s.count - j >= 32 ? 0xffffffffu : (1u << (s.count - j)) - 1u)) return true;
  return false;
}

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

// The 8 mask bits of node i from node j on.
__device__ __forceinline__ uint32_t node_mask(const AttendArgs &a, int b, int i, int j) {
  return j < a.rows ? a.mask[(size_t)b * a.mask_stride + (size_t)i * a.words + j / 32] >> (j % 32) : 0u;
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

// 4 f16 values of column m of the 16 lanes' 4 x 16 matrix, 4 values of a row at each of the lanes' addresses.
__device__ __forceinline__ u32x2 read_tr(const uint32_t *p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4 *)(__attribute__((address_space(3))) void *)p));
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

// Attention over a run of key blocks, for few rows.  A workgroup takes one key head of a sequence, 16 * QT of its rows
// (the heads / kv_heads query heads of a node are rows next to each other) and one split of its key blocks
// (64 positions for heads of up to 64 values, 32 for larger ones and of nodes), of which each of its kw wavefronts takes every
// kw-th.  A wavefront reads a block's K and V straight into the registers that the matrix cores take:
//
//   Scores transposed, S^T = K Q^T (v_mfma_f32_16x16x32_f16).  The cache holds K as pairs of values, position by
//   position, so a lane reads KP = 4 or 2 positions of a pair at once: lane 16g + m holds the positions from KP m on
//   of the pairs of 8 values from 8g on, which are the operand rows of KP tiles, tile u with position KP m + u in
//   row m.  In the products, lane 16g + i then holds row i's scores of the NP = 4 KP positions from NP g on.
//   Outputs transposed, O^T = V^T P^T: those scores are the operand of P as they stand, k = 8g + e of instruction kk
//   meaning position NP g + 8kk + e.  A lane reads 4 values (from 4m on) of its NP positions of V, and v_perm
//   pairs those of two positions.  A row's softmax state is one lane column's everywhere.
//
// The next block's K is asked for as soon as this one's scores are done, and its V after this one's outputs; the first
// block's before the queries are looked at.  For heads of 128 values this keeps loads in flight all the time.  In the code
// made for heads of up to 64, and of any size that is no multiple of 32, it does not: load_k's whole and partial chunks
// meet in the same registers, and each chunk's loads stand behind a wait for all that are under way, so that a block pays
// a round trip per chunk of K and one for V.  Both forms' addresses also cost 37 to 126 scalar registers kept in lanes of
// vector ones.  Bound by the cache's bytes where it is long (4 requests' 4 rows over 28 k keys of 8 heads of 128 values
// 85 us, 5.4 TB/s) and by that chain of loads where it is short (16 rows of 20 heads of 64 values over 391 keys: 7.6 us of
// kernel; 4 requests' 13 rows over 1100 to 1500: 11.4 us, twice their bytes' time).
//
// Precision: f32 queries are scaled by a power of two per row and split into two f16 parts, as is every
// softmax weight for f32 outputs: two products each, with an error of 2^-22 against f32's own 2^-24 per sum.  Weights
// are exp2(s - max + 10), so that the second part is no subnormal; a maximum that grows by less than SLACK binary
// digits is left as it is, since they still fit f16 then.  K and V are f16 as stored.
// P16 (f16 outputs): a weight is its first part alone, off by up to 2^-11 of itself, while the weights' sum stays f32.  Of 16
// requests' 61 f16 rows, values of 0.24, that makes the outputs' error 6.2e-5 (root mean square) where rounding them once
// leaves 5.0e-5; with both parts it is 5.0e-5 as well, and takes 16.4 us against 15.4 (4 requests' 100 rows over 28 k keys:
// 1.00e-5, 0.82e-5, and 120 us against 114).
//
// ONCE: the cache is read past the chip's own caches.
template <typename T, int HD, int QT, bool P16, bool ONCE>
__global__ __launch_bounds__(64 * WAVES) void attend_kernel(AttendArgs a) {
  constexpr int C = HD / 32, Z = HD / 64, QP = sizeof(T) == 4 ? 2 : 1;
  constexpr int KPC = few_block(HD) / 16, KB = 16 * KPC;
  typedef uint32_t Words __attribute__((ext_vector_type(KPC)));
  typedef Words Words_a4 __attribute__((aligned(4)));
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = threadIdx.x & 63, ki = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, m = lane & 15;
  const int split = blockIdx.z, kh = blockIdx.x, b = a.row_blocks == 1 ? blockIdx.y : blockIdx.y / a.row_blocks;
  const int group = a.heads / a.kv_heads, r0 = 16 * QT * (blockIdx.y - b * a.row_blocks);
  const size_t row0 = (size_t)b * a.rows;
  float f[QT][C][8];
  int node[QT];
#pragma unroll
  for (int t = 0; t < QT; t++) {  // (of rows that are not there, too: nothing is known of the lengths yet)
    const int row = min(r0 + 16 * t + m, a.rows * group - 1);
    node[t] = node_of(row, group);
    load_query<T, C>((const T *)a.q + (row0 + node[t]) * a.stride + (size_t)(kh * group + head_of(row, group)) * a.hd, g, a.hd, f[t]);
  }
  const Share s = share_of(a, b);
  const int total = s.count * group;
  if (split >= s.used || r0 >= total) return;
  const int half = a.kv_heads * a.hd / 2, pairs = a.hd / 2;
  const uint32_t *kc = a.kv + (size_t)b * a.kv_stride + (size_t)kh * pairs * a.cols;
  const uint32_t *vc = a.kv + (size_t)b * a.kv_stride + (size_t)half * a.cols + kh * pairs;

  Words kw[C][4];
  u32x2 vw[4 * KPC][Z];  // a block's K, pair by pair, and V, position by position
  auto load_k = [&](int blk) {
    // (made anew for every block: what follows from them would otherwise be kept in more registers than there are)
    int hd = a.hd, cols = a.cols;
    asm volatile("" : "+s"(hd), "+s"(cols));
    const int j0 = blk * KB, last = s.n - 1 - j0, jk = min(KPC * m, last & ~(KPC - 1));  // (a position past the row's end: the next row, or V)
#pragma unroll
    for (int c = 0; c < C; c++) {
      const uint32_t *base = kc + (size_t)(16 * c) * cols + j0;
      const int top = hd / 2 - 1 - 16 * c;  // the last pair of this chunk, where it has not 16
      if (top >= 15) {
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const Words_a4 *p = (const Words_a4 *)(base + (size_t)x * cols + (uint32_t)(4 * g * cols + jk));
          if constexpr (ONCE) kw[c][x] = __builtin_nontemporal_load(p);
          else kw[c][x] = *p;
        }
      } else {
#pragma unroll
        for (int x = 0; x < 4; x++) {
          kw[c][x] = *(const Words_a4 *)(base + (int64_t)max(min(4 * g + x, top), -16 * c) * cols + jk);
          if (top < 4 * g + x) kw[c][x] = Words{};
        }
      }
    }
  };
  auto load_v = [&](int blk) {
    const int j0 = blk * KB, last = s.n - 1 - j0;
    const uint32_t *base = vc + (size_t)j0 * half;
#pragma unroll
    for (int e = 0; e < 4 * KPC; e++)
#pragma unroll
      for (int z = 0; z < Z; z++) {
        const u32x2_a4 *p = (const u32x2_a4 *)(base + (uint32_t)(min(4 * KPC * g + e, last) * half + (64 * z + 4 * m < a.hd ? 32 * z + 2 * m : 0)));
        if constexpr (ONCE) vw[e][z] = __builtin_nontemporal_load(p);
        else vw[e][z] = *p;
      }
  };
  auto load_nodes = [&](int blk) {
    const int j0 = (blk - s.cached) * NODES, last = s.count - 1 - j0;
    const T *k = (const T *)a.k + (row0 + j0) * a.stride + (size_t)kh * a.hd;
    const T *v = (const T *)a.v + (row0 + j0) * a.stride + (size_t)kh * a.hd;
    // (every row's loads before the first one is rounded; larger heads' K first and then V, for want of registers)
    typename Four<T>::type rk[C][2][2], rv[8][Z];
    auto round_k = [&] {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int y = 0; y < 2; y++) {
            const u32x2 w = 32 * c + 8 * g + 4 * y < a.hd ? pairs4(rk[c][u][y]) : u32x2{};
            kw[c][2 * y][u] = w[0], kw[c][2 * y + 1][u] = w[1];
          }
    };
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int y = 0; y < 2; y++) {
          const int d = 32 * c + 8 * g + 4 * y;
          rk[c][u][y] = raw4(k + (uint32_t)min(2 * m + u, last) * (uint32_t)a.stride + (d < a.hd ? d : 0));
        }
    if constexpr (Z == 2) round_k();
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int z = 0; z < Z; z++)
        rv[e][z] = raw4(v + (uint32_t)min(8 * g + e, last) * (uint32_t)a.stride + (64 * z + 4 * m < a.hd ? 64 * z + 4 * m : 0));
    if constexpr (Z == 1) round_k();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int z = 0; z < Z; z++) vw[e][z] = pairs4(rv[e][z]);
  };
  int blk = split * s.per + ki;
  const int end = min((split + 1) * s.per, s.blocks), cached = min(end, s.cached);
  if (blk < cached) {
    if (a.cols >= KPC) {
      load_k(blk);
    } else {  // (a cache of so few positions: nothing behind them)
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
          for (int u = 0; u < KPC; u++) {
            const int p = 16 * c + 4 * g + x;
            kw[c][x][u] = p < pairs ? kc[p * a.cols + min(u, a.cols - 1)] : 0u;
          }
    }
    load_v(blk);
  } else if (blk < end) {
    load_nodes(blk);
  }

  half8 q[QT][C][QP];
  floatx4 acc[QT][4 * Z];
  float mx[QT], sum[QT], cf[QT], slack[QT];
#pragma unroll
  for (int t = 0; t < QT; t++) {
    cf[t] = split_query(f[t], a.scale, q[t]);
    if (r0 + 16 * t + m >= total) cf[t] = 0.0f;  // (whatever stands in a row past the last: no maximum, no far score)
    slack[t] = SLACK / cf[t];
    mx[t] = -INFINITY, sum[t] = 0.0f;
#pragma unroll
    for (int x = 0; x < 4 * Z; x++) acc[t][x] = floatx4{};
  }
  // One block: 0 a whole one of the cache, with the next one's loads; 1 the last one of the cache; 2 one of nodes.
  auto step = [&](auto which) {
    constexpr int KIND = which;
    constexpr bool all = KIND == 0;
    constexpr int KP = KIND == 2 ? 2 : KPC, NP = 4 * KP, KK = KP / 2;
    const int j0 = KIND == 2 ? (blk - s.cached) * NODES : blk * KB, last = (KIND == 2 ? s.count : s.n) - 1 - j0;
    const int left = last + 1 - NP * g;  // of this lane's positions
    floatx4 st[QT][KP];
#pragma unroll
    for (int t = 0; t < QT; t++)
#pragma unroll
      for (int u = 0; u < KP; u++) st[t][u] = floatx4{};
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int u = 0; u < KP; u++) {
        const half8 k = __builtin_bit_cast(half8, u32x4{kw[c][0][u], kw[c][1][u], kw[c][2][u], kw[c][3][u]});
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int part = 0; part < QP; part++) st[t][u] = mfma(k, q[t][c][part], st[t][u]);
      }
    if constexpr (KIND == 0) load_k(blk + a.kw);

    // The softmax: element KP r + u of the lane's NP positions is st[u][r].
    if constexpr (!all) {
      const uint32_t there = left >= NP ? (1u << NP) - 1u : left > 0 ? (1u << left) - 1u : 0u;
#pragma unroll
      for (int t = 0; t < QT; t++) {
        uint32_t vis = there;
        if constexpr (KIND == 2) vis &= node_mask(a, b, node[t], j0 + NP * g);
#pragma unroll
        for (int e = 0; e < NP; e++)
          if (!(vis >> e & 1)) st[t][e % KP][e / KP] = -INFINITY;
      }
    }
    half8 ph[QT][KK], pl[QT][KK];
#pragma unroll
    for (int t = 0; t < QT; t++) {
      float top = st[t][0][0];
#pragma unroll
      for (int e = 1; e < NP; e++) top = fmaxf(top, st[t][e % KP][e / KP]);
      top = xlane::bit4(top, xlane::Max{});
      top = xlane::bit5(top, xlane::Max{});
      if (__any(top > mx[t] + slack[t])) {
        top = fmaxf(top, mx[t]);
        const float old = mx[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mx[t] - top) * cf[t]);
        sum[t] *= old;
#pragma unroll
        for (int x = 0; x < 4 * Z; x++) acc[t][x] *= old;
        mx[t] = top;
      }
      const float base = mx[t] == -INFINITY ? 0.0f : mx[t];
      float shift = fmaf(-base, cf[t], 10.0f);
      if (__any(fabsf(shift) > FAR)) {
        shift = 10.0f;
#pragma unroll
        for (int u = 0; u < KP; u++) st[t][u] -= base;
      }
#pragma unroll
      for (int e = 0; e < NP; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(st[t][e % KP][e / KP], cf[t], shift));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(st[t][(e + 1) % KP][(e + 1) / KP], cf[t], shift));
        sum[t] += p0, sum[t] += p1;
        weights2<P16>(p0, p1, ph[t][e >> 3], pl[t][e >> 3], e & 7);
      }
    }

    if constexpr (!all) {
      // Values of positions that are not there are zeroed, and so are a node's that are no finite numbers: those must not
      // meet the zero weights of the rows that do not see them, and are added to the others' outputs one by one.
      u16x2 big{};
#pragma unroll
      for (int e = 0; e < NP; e++)
#pragma unroll
        for (int z = 0; z < Z; z++) {
          if (e >= left) vw[e][z] = u32x2{};
          if constexpr (KIND != 2) continue;
          big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, vw[e][z][0] & 0x7fff7fffu));
          big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, vw[e][z][1] & 0x7fff7fffu));
        }
      if (KIND == 2 && __any(big[0] >= 0x7c00 || big[1] >= 0x7c00)) {
#pragma unroll
        for (int e = 0; e < NP; e++)
#pragma unroll
          for (int z = 0; z < Z; z++) vw[e][z] = u32x2{finite2(vw[e][z][0]), finite2(vw[e][z][1])};
#pragma unroll 1
        for (int j = 0; j < min(NODES, last + 1); j++) {
          int hd = a.hd;
          asm volatile("" : "+s"(hd));  // (nothing of this loop is worth a register outside)
          const T *v = (const T *)a.v + (row0 + j0 + j) * a.stride + (size_t)kh * a.hd;
#pragma unroll
          for (int t = 0; t < QT; t++) {
            if (!(node_mask(a, b, node[t], j0 + j) & 1)) continue;
#pragma unroll
            for (int x = 0; x < 4 * Z; x++)
#pragma unroll
              for (int r = 0; r < 4; r++) acc[t][x][r] += not_finite(v, 64 * (x / 4) + 16 * g + 4 * r + x % 4, hd);
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 4 * Z; x++)
#pragma unroll
      for (int kk = 0; kk < KK; kk++) {
        u32x4 w;
#pragma unroll
        for (int y = 0; y < 4; y++)
          w[y] = __builtin_amdgcn_perm(vw[8 * kk + 2 * y + 1][x / 4][x % 4 / 2], vw[8 * kk + 2 * y][x / 4][x % 4 / 2],
                                       x & 1 ? 0x07060302u : 0x05040100u);
        const half8 vf = __builtin_bit_cast(half8, w);
#pragma unroll
        for (int t = 0; t < QT; t++) {
          acc[t][x] = mfma(vf, ph[t][kk], acc[t][x]);
          if constexpr (!P16) acc[t][x] = mfma(vf, pl[t][kk], acc[t][x]);
        }
      }
    if constexpr (KIND == 0) load_v(blk + a.kw);
  };
  bool loaded = true;
  if (blk < cached) {
    for (; blk + a.kw < cached; blk += a.kw) step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    blk += a.kw, loaded = false;
  }
  for (; blk < end; blk += a.kw, loaded = false) {
    if (!loaded) load_nodes(blk);
    step(std::integral_constant<int, 2>{});
  }

  // The wavefronts' results joined through LDS: each writes its own, then every lane adds up four values of a row, all of
  // its reads at once.  Lane 16g + i holds row i's values 16g + 4r + (x % 4) of the chunk of 64 x / 4.
  floatx4 *merge = (floatx4 *)smem;                       // [ki][t][z][r][lane]
  float *ml = (float *)(merge + a.kw * QT * Z * 256);  // [ki][t][maxima, sums][row]
#pragma unroll
  for (int t = 0; t < QT; t++) {
    sum[t] = xlane::bit4(sum[t], xlane::Add{});
    sum[t] = xlane::bit5(sum[t], xlane::Add{});
    if (g == 0) ml[32 * (ki * QT + t) + m] = mx[t], ml[32 * (ki * QT + t) + 16 + m] = sum[t];
#pragma unroll
    for (int z = 0; z < Z; z++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        merge[(((ki * QT + t) * Z + z) * 4 + r) * 64 + lane] =
            floatx4{acc[t][4 * z][r], acc[t][4 * z + 1][r], acc[t][4 * z + 2][r], acc[t][4 * z + 3][r]};
  }
  __syncthreads();
  for (int x = ki; x < QT * Z * 4; x += a.kw) {
    const int t = x / (4 * Z), z = x / 4 % Z, d = 64 * z + 16 * g + 4 * (x % 4), r = r0 + 16 * t + m;
    if (r >= total || d >= a.hd) continue;
    float km[WAVES], kl[WAVES], top = -INFINITY, l = 0.0f, c = cf[0];
    if (QT == 2 && t) c = cf[QT - 1];
    floatx4 kf[WAVES], f{};
#pragma unroll
    for (int k = 0; k < WAVES; k++) {
      const int w = min(k, a.kw - 1) * QT;
      km[k] = ml[32 * (w + t) + m], kl[k] = ml[32 * (w + t) + 16 + m], kf[k] = merge[(w * Z * 4 + x) * 64 + lane];
      if (k >= a.kw) km[k] = -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < WAVES; k++) top = fmaxf(top, km[k]);
#pragma unroll
    for (int k = 0; k < WAVES; k++) {
      if (k >= a.kw) break;
      const float w = km[k] == top ? 1.0f : __builtin_amdgcn_exp2f((km[k] - top) * c);
      l += w * kl[k], f += w * kf[k];
    }
    const int i = node_of(r, group), head = kh * group + head_of(r, group);
    const size_t out = ((row0 + i) * a.heads + head) * a.hd + d;
    if (s.used > 1) {
      const size_t part = (size_t)split * a.batch * a.rows * a.heads;
      if (d == 0) *(floatx4 *)(a.pml + 4 * (part + (row0 + i) * a.heads + head)) = floatx4{top, l, c, 0.0f};
      *(floatx4 *)(a.po + part * a.hd + out) = f;
      continue;
    }
    f *= l == 0.0f && !sees_any(a, s, b, i) ? 0.0f : 1.0f / l;
    if constexpr (P16) *(u32x2_a4 *)((_Float16 *)a.o + out) = u32x2{pack2(f[0], f[1]), pack2(f[2], f[3])};
    else *(floatx4_a4 *)((float *)a.o + out) = f;
  }
}

// The same for more rows of a key head: a workgroup's RT wavefronts have 16 rows each and go through the key blocks
// (64 positions for heads of up to 64 values, 32 for larger ones: 16 KiB) one after the other.  Its threads load a
// block two blocks ahead, each its share of 16-byte pieces, and write it to one of two LDS buffers, K position by
// position too, from which the wavefronts read operands as they stand: 8 values of a position of K, and V
// transposed by ds_read_b64_tr_b16 (rows 16 and 32 bytes longer, for the banks' sake).  Tile u's row r is position
// 16u + r, so lane 16g + i's scores are those of positions 16u + 4g + 0 .. 3 of every u.  Workgroups of 8 wavefronts
// get by with 128 registers, so that two share a CU, those of 4 with 168 for three; f32 queries of heads past 64 values need 8
// more than the former 128, which are spilled outside the loop over the cache.  Its wavefronts wait for each other
// block by block, so the matrix cores, LDS and the softmax's instructions share the time rather than overlap (200 rows of
// f32 queries on 64 values over 23 k keys: vector instructions 50 % of it, matrix cores 29 %): 4 requests' 100 f16 rows over 28 k keys of
// 8 heads of 128 values 114 us (4.0 TB/s, 305 TFLOP/s), 16 requests' 61 rows over up to 448 keys of 20 heads 15.4 us.
// The nodes' rows and masks are asked for only when the cache's blocks are done, which such short caches feel.
template <typename T, int HD, int RT, bool P16>
__global__ __launch_bounds__(64 * RT, RT == 8 ? 4 : 3) void attend_rows_kernel(AttendArgs a) {
  constexpr int C = HD / 32, X = HD / 16, QP = sizeof(T) == 4 ? 2 : 1, B = rows_block(HD), NT = B / 16, KK = B / 32;
  constexpr int KS = HD / 2 + 4, VS = HD / 2 + 8;  // words per position of K and of V in LDS
  constexpr int KW = KS * B, BUF = KW + VS * B, U = 512;  // words of K and of a buffer; 16-byte pieces of K or V
  extern __shared__ __attribute__((aligned(16))) uint32_t words[];
  __shared__ int odd;  // set where a node's value is no finite number
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, m = lane & 15;
  const int tid = threadIdx.x;
  constexpr int threads = 64 * RT, MOST = U / threads;  // MOST: pieces per thread
  const int split = blockIdx.z, kh = blockIdx.x, b = a.row_blocks == 1 ? blockIdx.y : blockIdx.y / a.row_blocks;
  const int rb = blockIdx.y - b * a.row_blocks;
  const int group = a.heads / a.kv_heads, r0 = 16 * (rb * RT + wave);
  const size_t row0 = (size_t)b * a.rows;
  const Share s = share_of(a, b);
  const int total = s.count * group;
  if (split >= s.used || 16 * RT * rb >= total) return;
  const int half = a.kv_heads * a.hd / 2, pairs = a.hd / 2;
  const uint32_t *kc = a.kv + (size_t)b * a.kv_stride + (size_t)kh * pairs * a.cols;
  const uint32_t *vc = a.kv + (size_t)b * a.kv_stride + (size_t)half * a.cols + kh * pairs;
  const int begin = split * s.per, end = min(begin + s.per, s.blocks), cached = min(end, s.cached);

  // A cached block's pieces into registers, then into LDS.
  struct Pieces {
    u32x4 k[MOST], v[MOST];
  };
  // Piece u of K: 4 positions from 4q on of a pair, 4 such next to each other in memory and 16 pairs per wavefront, so that
  // a position's words go to different banks; of V: 8 values of a position.
  uint32_t kat[MOST], vat[MOST];  // words from the block's first ones
  int kq[MOST], kpair[MOST], vrow[MOST], vd[MOST];
#pragma unroll
  for (int i = 0; i < MOST; i++) {
    const int u = tid + threads * i;
    kq[i] = 4 * (u % 4 + 4 * (u / 64 % (B / 16))), kpair[i] = u % 64 / 4 + 16 * (u / 64 / (B / 16));
    vrow[i] = u / (HD / 8), vd[i] = u % (HD / 8) * 4;
    kat[i] = (uint32_t)min(kpair[i], pairs - 1) * (uint32_t)a.cols, vat[i] = (uint32_t)min(vd[i], pairs - 4);
  }
  auto load = [&](Pieces &p, int blk) {
    const int j0 = blk * B, last = s.n - 1 - j0;
    const bool inside = j0 + B <= a.cols;  // (positions past n are there to be read, at least)
    const uint32_t *kb = kc + j0, *vb = vc + (size_t)j0 * half;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      p.k[i] = *(const u32x4_a4 *)(kb + (kat[i] + (inside ? kq[i] : min(kq[i], last & ~3))));
      p.v[i] = *(const u32x4_a4 *)(vb + (vat[i] + (inside ? vrow[i] : min(vrow[i], last)) * half));
    }
  };
  auto store = [&](const Pieces &p, int blk, uint32_t *buf) {
    const int last = s.n - 1 - blk * B;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      u32x4 k = p.k[i], v = p.v[i];
      if (a.hd < HD) {  // (a head's last 4 values can be the upper half of the piece before its end)
        if (kpair[i] >= pairs) k = u32x4{};
        if (vd[i] == pairs - 2) v = u32x4{v[2], v[3], 0, 0};
      }
      if (last < B - 1 && vrow[i] > last) v = u32x4{};
#pragma unroll
      for (int e = 0; e < 4; e++) buf[(kq[i] + e) * KS + kpair[i]] = k[e];
      *(u32x4 *)(buf + KW + vrow[i] * VS + vd[i]) = v;
    }
  };
  Pieces p0, p1;
  int blk = begin;
  if (blk < cached) load(p0, blk);
  if (blk + 1 < cached) load(p1, blk + 1);

  half8 q[C][QP];
  floatx4 acc[X];
  float mx = -INFINITY, sum = 0.0f;
  const int row = min(r0 + m, total - 1), node = node_of(row, group), head = kh * group + head_of(row, group);
  float f[C][8];
  load_query<T, C>((const T *)a.q + (row0 + node) * a.stride + (size_t)head * a.hd, g, a.hd, f);
  const float cf = split_query(f, a.scale, q), slack = SLACK / cf;
#pragma unroll
  for (int x = 0; x < X; x++) acc[x] = floatx4{};
  const bool busy = r0 < total;  // (a wavefront past the last row only loads)

  // One block from LDS; nodes: a block of nodes, otherwise the cache's.
  auto step = [&](auto nodes, int blk, const uint32_t *buf) {
    constexpr bool NODES = nodes;
    const int j0 = (NODES ? blk - s.cached : blk) * B, last = (NODES ? s.count : s.n) - 1 - j0;
    floatx4 st[NT];
#pragma unroll
    for (int u = 0; u < NT; u++) st[u] = floatx4{};
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int u = 0; u < NT; u++) {
        const half8 kf = *(const half8 *)(buf + (16 * u + m) * KS + 16 * c + 4 * g);
#pragma unroll
        for (int part = 0; part < QP; part++) st[u] = mfma(kf, q[c][part], st[u]);
      }
    if (NODES || last < B - 1) {
#pragma unroll
      for (int kk = 0; kk < KK; kk++) {
        const int left = last + 1 - 32 * kk;
        uint32_t vis = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
        if constexpr (NODES) vis &= node_mask(a, b, node, j0 + 32 * kk);
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (!(vis >> (16 * (e >> 2) + 4 * g + (e & 3)) & 1)) st[2 * kk + (e >> 2)][e & 3] = -INFINITY;
      }
    }
    // V's operands are read a step ahead of their products.
    half8 vf[2][KK];
    auto read_v = [&](int x) {
#pragma unroll
      for (int kk = 0; kk < KK; kk++) {
        const uint32_t *v = buf + KW + (32 * kk + 4 * g + (m >> 2)) * VS + 8 * x + 2 * (m & 3);
        const u32x2 lo = read_tr(v), hi = read_tr(v + 16 * VS);
        vf[x & 1][kk] = __builtin_bit_cast(half8, u32x4{lo[0], lo[1], hi[0], hi[1]});
      }
    };
    read_v(0);
    half8 ph[KK], pl[KK];
    float top = st[0][0];
#pragma unroll
    for (int e = 1; e < 4 * NT; e++) top = fmaxf(top, st[e >> 2][e & 3]);
    top = xlane::bit4(top, xlane::Max{});
    top = xlane::bit5(top, xlane::Max{});
    if (__any(top > mx + slack)) {
      top = fmaxf(top, mx);
      const float old = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mx - top) * cf);
      sum *= old;
#pragma unroll
      for (int x = 0; x < X; x++) acc[x] *= old;
      mx = top;
    }
    const float base = mx == -INFINITY ? 0.0f : mx;
    float shift = fmaf(-base, cf, 10.0f);
    if (__any(fabsf(shift) > FAR)) {
      shift = 10.0f;
#pragma unroll
      for (int u = 0; u < NT; u++) st[u] -= base;
    }
#pragma unroll
    for (int e = 0; e < 4 * NT; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(st[e >> 2][e & 3], cf, shift));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(st[e >> 2][(e + 1) & 3], cf, shift));
      sum += p0, sum += p1;
      weights2<P16>(p0, p1, ph[e >> 3], pl[e >> 3], e & 7);
    }
#pragma unroll
    for (int x = 0; x < X; x++) {
      if (x + 1 < X) read_v(x + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < KK; kk++) {
        acc[x] = mfma(vf[x & 1][kk], ph[kk], acc[x]);
        if constexpr (!P16) acc[x] = mfma(vf[x & 1][kk], pl[kk], acc[x]);
      }
    }
    if (NODES && odd)  // what the block has zeros for, to the rows that see it
#pragma unroll 1
      for (int j = 0; j < min(B, last + 1); j++) {
        int hd = a.hd;
        asm volatile("" : "+s"(hd));
        if (!(node_mask(a, b, node, j0 + j) & 1)) continue;
        const T *v = (const T *)a.v + (row0 + j0 + j) * a.stride + (size_t)kh * a.hd;
#pragma unroll
        for (int x = 0; x < X; x++)
#pragma unroll
          for (int r = 0; r < 4; r++) acc[x][r] += not_finite(v, 16 * x + 4 * g + r, hd);
      }
  };

  // The blocks pass in turn through p0 and the first buffer and through p1 and the second.  A buffer is written again
  // two blocks later, past the barrier that every wavefront reaches after it has read it.
  uint32_t *const buf0 = words, *const buf1 = buf0 + BUF;
  for (; blk + 4 <= cached; blk += 2) {
    store(p0, blk, buf0);
    load(p0, blk + 2);
    meet();
    if (busy) step(std::false_type{}, blk, buf0);
    store(p1, blk + 1, buf1);
    load(p1, blk + 3);
    meet();
    if (busy) step(std::false_type{}, blk + 1, buf1);
  }
  for (bool even = true; blk < cached; blk++, even = !even) {  // (three at most)
    if (even) {
      store(p0, blk, buf0);
      if (blk + 2 < cached) load(p0, blk + 2);
    } else {
      store(p1, blk, buf1);
    }
    meet();
    if (busy) step(std::false_type{}, blk, even ? buf0 : buf1);
  }
  for (; blk < end; blk++) {
    const int j0 = (blk - s.cached) * B, last = s.count - 1 - j0;
    __syncthreads();
    if (tid == 0) odd = 0;
    __syncthreads();
    bool found = false;
    typename Four<T>::type rk[MOST][2], rv[MOST][2];  // (every row's loads before the first one is rounded)
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int u = tid + threads * i, row = u / (HD / 8), d = u % (HD / 8) * 8;
      const size_t src = (row0 + j0 + min(row, last)) * a.stride + (size_t)kh * a.hd;
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const int at = d + 4 * y < a.hd ? d + 4 * y : 0;
        rk[i][y] = raw4((const T *)a.k + src + at), rv[i][y] = raw4((const T *)a.v + src + at);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int u = tid + threads * i, row = u / (HD / 8), d = u % (HD / 8) * 8;
      u32x2 k[2], v[2];
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const bool in = d + 4 * y < a.hd;
        k[y] = in ? pairs4(rk[i][y]) : u32x2{}, v[y] = in && row <= last ? pairs4(rv[i][y]) : u32x2{};
        const u32x2 clean{finite2(v[y][0]), finite2(v[y][1])};
        found |= clean[0] != v[y][0] || clean[1] != v[y][1];
        v[y] = clean;
      }
      *(u32x4 *)(buf0 + row * KS + d / 2) = u32x4{k[0][0], k[0][1], k[1][0], k[1][1]};
      *(u32x4 *)(buf0 + KW + row * VS + d / 2) = u32x4{v[0][0], v[0][1], v[1][0], v[1][1]};
    }
    if (found) odd = 1;
    __syncthreads();
    if (busy) step(std::true_type{}, blk, buf0);
  }

  sum = xlane::bit4(sum, xlane::Add{});
  sum = xlane::bit5(sum, xlane::Add{});
  if (r0 + m >= total) return;
  // Lane 16g + i holds row i's values 16x + 4g + 0 .. 3.
  const size_t out = ((row0 + node) * a.heads + head) * a.hd, part = (size_t)split * a.batch * a.rows * a.heads;
  if (s.used > 1 && g == 0) *(floatx4 *)(a.pml + 4 * (part + (row0 + node) * a.heads + head)) = floatx4{mx, sum, cf, 0.0f};
  const float inv = s.used > 1 ? 1.0f : sum == 0.0f && !sees_any(a, s, b, node) ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int x = 0; x < X; x++) {
    const int d = 16 * x + 4 * g;
    if (d >= a.hd) continue;
    const floatx4 o = acc[x] * inv;
    if (s.used > 1) *(floatx4 *)(a.po + part * a.hd + out + d) = o;
    else if constexpr (P16) *(u32x2_a4 *)((_Float16 *)a.o + out + d) = u32x2{pack2(o[0], o[1]), pack2(o[2], o[3])};
    else *(floatx4_a4 *)((float *)a.o + out + d) = o;
  }
}

// The splits' outputs of one head of a node rescaled to their common maximum, summed and divided; one wavefront
// each: split x's maximum and sum in lane x, then two values a lane, 8 splits' at a time.
constexpr int SPLITS = 64;

template <bool P16>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a) {
  const int lane = threadIdx.x & 63, at = blockIdx.x * 4 + (threadIdx.x >> 6), heads = a.batch * a.rows * a.heads;
  if (at >= heads) return;
  const int row = at / a.heads, b = row / a.rows, i = row % a.rows;
  const Share s = share_of(a, b);
  if (s.used == 1 || i >= s.count) return;
  const floatx4 ml = *(const floatx4 *)(a.pml + 4 * ((size_t)min(lane, s.used - 1) * heads + at));
  const bool mine = lane < s.used;
  const float top = xlane::wave_max(mine ? ml[0] : -INFINITY);
  const float w = !mine ? 0.0f : ml[0] == top ? 1.0f : __builtin_amdgcn_exp2f((ml[0] - top) * ml[2]);
  const float sum = xlane::wave_sum(mine ? w * ml[1] : 0.0f);
  const int d = min(2 * lane, a.hd - 2);
  float o0 = 0.0f, o1 = 0.0f;
  for (int x = 0; x < s.used; x += 8) {
    float2 p[8];
#pragma unroll
    for (int y = 0; y < 8; y++) p[y] = *(const float2 *)(a.po + ((size_t)min(x + y, s.used - 1) * heads + at) * a.hd + d);
#pragma unroll
    for (int y = 0; y < 8; y++) {
      const float f = __shfl(w, x + y);
      if (x + y < s.used) o0 += f * p[y].x, o1 += f * p[y].y;
    }
  }
  if (2 * lane >= a.hd) return;
  const float inv = sum == 0.0f && !sees_any(a, s, b, i) ? 0.0f : 1.0f / sum;
  if constexpr (P16) {
    *(uint32_t *)((_Float16 *)a.o + (size_t)at * a.hd + d) = pack2(o0 * inv, o1 * inv);
  } else {
    float *o = (float *)a.o + (size_t)at * a.hd + d;
    o[0] = o0 * inv, o[1] = o1 * inv;
  }
}

// ------------------------------------------------------------------------------------- the kept path

struct AcceptArgs {
  const int32_t *n, *count;
  const uint32_t *tokens, *mask, *picks;
  size_t mask_stride;
  int rows, words, cols;
  int32_t *path, *kept;
  uint32_t *next;
  int32_t *n_out;
  uint32_t *history;
  int history_cols;
};

// The walk of sequence b, by a whole workgroup: every node's parent (the highest bit below its own) and whether its
// token is the parent's pick; of a parent's agreeing children the first; then from the root on.  path: LDS.
__device__ __forceinline__ int walk(const AcceptArgs &a, int b, int n, int count, int *child, int *path, int *kept) {
  const int tid = threadIdx.x;
  const uint32_t *tokens = a.tokens + (size_t)b * a.rows, *picks = a.picks + (size_t)b * a.rows;
  for (int i = tid; i < count; i += 256) child[i] = INT_MAX;
  __syncthreads();
  for (int i = 1 + tid; i < count; i += 256) {
    const uint32_t *w = a.mask + (size_t)b * a.mask_stride + (size_t)i * a.words;
    int parent = -1;
    for (int x = i / 32; x >= 0 && parent < 0; x--) {
      const uint32_t bits = x == i / 32 ? w[x] & ((1u << (i % 32)) - 1u) : w[x];
      if (bits) parent = 32 * x + 31 - __clz((int)bits);
    }
    if (parent >= 0 && picks[parent] != 0xffffffffu && tokens[i] == picks[parent]) atomicMin(&child[parent], i);
  }
  __syncthreads();
  if (tid == 0) {
    int room = a.cols - n;
    if (a.history) room = min(room, a.history_cols - n);
    int k = 0;
    for (int i = 0; i < count && k < room; i = child[i]) path[k++] = i;
    *kept = k;
  }
  __syncthreads();
  return *kept;
}

// What the walk says of sequence b.
__device__ __forceinline__ void tell(const AcceptArgs &a, int b, int n, int count, const int *path, int kept) {
  const int tid = threadIdx.x;
  const uint32_t *tokens = a.tokens + (size_t)b * a.rows, *picks = a.picks + (size_t)b * a.rows;
  for (int i = tid; i < a.rows; i += 256) a.path[(size_t)b * a.rows + i] = i < kept ? path[i] : -1;
  if (a.history)
    for (int i = tid; i < kept; i += 256) a.history[(size_t)b * a.history_cols + n + i] = tokens[path[i]];
  __syncthreads();  // (next may be the tokens themselves, where a root is all there is)
  if (tid == 0) {
    a.kept[b] = kept;
    a.n_out[b] = n + kept;
    if (count) a.next[b] = kept ? picks[path[kept - 1]] : tokens[0];
  }
}

__global__ __launch_bounds__(256) void accept_kernel(AcceptArgs a) {
  __shared__ int child[TREE_ROWS], path[TREE_ROWS], kept;
  const int b = blockIdx.x, n = min(max(a.n[b], 0), a.cols), count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows;
  const int k = walk(a, b, n, count, child, path, &kept);
  tell(a, b, n, count, path, k);
}

struct KeepArgs {
  const void *k, *v;
  size_t stride, layer_stride;
  uint32_t *kv;
  size_t kv_stride, kv_layer_stride;
  int d, parts;
  bool walks;  // the workgroups walk the trees themselves; otherwise the outputs are there
};

// The kept nodes' K and V into the caches: a thread per pair of values, K's pairs and then V's.  Bound by its chain of
// loads and by K's layout, whose words of a position lie `cols` apart: AT positions' rows are loaded side by side, and
// four neighbouring positions' words of a pair of K go in one store (9 nodes of 1280 values for 32 sequences and 4
// layers: 10.2 us of kernel, 1.7 TB/s; word by word 12.7).
template <typename T>
__global__ __launch_bounds__(256) void keep_kernel(AcceptArgs t, KeepArgs a) {
  typedef T Pair __attribute__((ext_vector_type(2)));
  typedef Pair any __attribute__((aligned(4)));
  typedef uint32_t Words __attribute__((ext_vector_type(4)));
  typedef Words words_at __attribute__((aligned(4)));
  constexpr int AT = 8;
  __shared__ int child[TREE_ROWS], path[TREE_ROWS], found;
  const int part = blockIdx.x % a.parts, b = blockIdx.x / a.parts, layer = blockIdx.y;
  int kept, n;
  if (a.walks) {
    n = min(max(t.n[b], 0), t.cols);
    const int count = t.count ? min(max(t.count[b], 0), t.rows) : t.rows;
    kept = walk(t, b, n, count, child, path, &found);
    if (part == 0 && layer == 0) tell(t, b, n, count, path, kept);
  } else {
    kept = t.kept[b], n = t.n_out[b] - kept;
    for (int i = threadIdx.x; i < kept; i += 256) path[i] = t.path[(size_t)b * t.rows + i];
    __syncthreads();
  }
  const int i = part * 256 + threadIdx.x, half = a.d / 2;
  if (i >= a.d) return;
  const int c = i < half ? i : i - half;
  const T *x = (const T *)(i < half ? a.k : a.v) + layer * a.layer_stride + (size_t)b * t.rows * a.stride + 2 * c;
  uint32_t *y = a.kv + layer * a.kv_layer_stride + b * a.kv_stride +
                (i < half ? (size_t)c * t.cols + n : (size_t)half * t.cols + (size_t)n * half + c);
  const size_t step = i < half ? 1 : half;
  for (int s = 0; s < kept; s += AT) {
    Pair p[AT];
#pragma unroll
    for (int e = 0; e < AT; e++) p[e] = *(const any *)(x + (size_t)path[min(s + e, kept - 1)] * a.stride);
#pragma unroll
    for (int e = 0; e < AT; e += 4) {
      Words w;
#pragma unroll
      for (int f = 0; f < 4; f++)
        w[f] = __builtin_bit_cast(uint16_t, (_Float16)p[e + f][0]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)p[e + f][1]) << 16;
      if (i < half && s + e + 4 <= kept) {
        *(words_at *)(y + s + e) = w;
      } else {
#pragma unroll
        for (int f = 0; f < 4; f++)
          if (s + e + f < kept) y[(s + e + f) * step] = w[f];
      }
    }
  }
}

template <typename T, int HD, int QT, bool P16>
int attend_launch(wh_ctx *ctx, const AttendArgs &a, bool once) {
  ProfScope prof(ctx, "tree_attend", 4.0 * a.batch * a.rows * a.heads * a.cols * a.hd, 4.0 * a.batch * a.cols * a.kv_heads * a.hd);
  const dim3 grid(a.kv_heads, a.batch * a.row_blocks, a.splits);
  const size_t shm = (size_t)a.kw * QT * (HD / 64 * 4096 + 128);
  if (once) wh_launch(ctx, (attend_kernel<T, HD, QT, P16, true>), grid, 64 * a.kw, shm, a);
  else wh_launch(ctx, (attend_kernel<T, HD, QT, P16, false>), grid, 64 * a.kw, shm, a);
  return wh_launched(ctx, "tree attention");
}

template <bool P16>
int attend_join(wh_ctx *ctx, const AttendArgs &a) {
  const double heads = (double)a.batch * a.rows * a.heads;
  ProfScope prof(ctx, "tree_attend_join", 0.0, 4.0 * heads * a.splits * (a.hd + 4));
  wh_launch(ctx, attend_join_kernel<P16>, (a.batch * a.rows * a.heads + 3) / 4, 256, 0, a);
  return wh_launched(ctx, "tree attention's join");
}

template <typename T, int HD, int RT, bool P16>
int attend_rows_launch(wh_ctx *ctx, const AttendArgs &a) {
  constexpr int B = rows_block(HD);
  ProfScope prof(ctx, "tree_attend_rows", 4.0 * a.batch * a.rows * a.heads * a.cols * a.hd, 4.0 * a.batch * a.cols * a.kv_heads * a.hd);
  wh_launch(ctx, (attend_rows_kernel<T, HD, RT, P16>), dim3(a.kv_heads, a.batch * a.row_blocks, a.splits), 64 * RT, 2 * 4 * (HD + 12) * B, a);
  return wh_launched(ctx, "tree attention");
}

// rt: row tiles of attend_rows_kernel's workgroups, or 0: attend_kernel with qt tiles of rows; once: see there.
template <typename T, bool P16>
int attend_t(wh_ctx *ctx, const AttendArgs &a, int qt, int rt, bool once) {
  int rc;
  if (rt && a.hd <= 64) rc = rt == 4 ? attend_rows_launch<T, 64, 4, P16>(ctx, a) : attend_rows_launch<T, 64, 8, P16>(ctx, a);
  else if (rt) rc = rt == 4 ? attend_rows_launch<T, 128, 4, P16>(ctx, a) : attend_rows_launch<T, 128, 8, P16>(ctx, a);
  else if (a.hd <= 64) rc = qt == 1 ? attend_launch<T, 64, 1, P16>(ctx, a, once) : attend_launch<T, 64, 2, P16>(ctx, a, once);
  else rc = attend_launch<T, 128, 1, P16>(ctx, a, once);
  return rc || a.splits == 1 ? rc : attend_join<P16>(ctx, a);
}

}  // namespace

int tree_check(wh_ctx *ctx, const char *what, const wh_tree *t) {
  if (!t || t->batch <= 0 || t->rows <= 0 || t->rows > TREE_ROWS || (size_t)t->batch * t->rows > TREE_NODES || !t->n)
    return wh_fail(ctx, WH_EARG, "%s: a tree of %d sequences of %d nodes (at most %d, %d in all) with lengths is needed", what,
                   t ? t->batch : 0, t ? t->rows : 0, TREE_ROWS, TREE_NODES);
  if (t->mask && t->mask_stride && t->mask_stride < (size_t)t->rows * ((t->rows + 31) / 32))
    return wh_fail(ctx, WH_EARG, "%s: masks %zu words apart, %d nodes take more", what, t->mask_stride, t->rows);
  if (((uintptr_t)t->n | (uintptr_t)t->count | (uintptr_t)t->tokens | (uintptr_t)t->mask) % 4)
    return wh_fail(ctx, WH_EARG, "%s: the tree's arrays must be 4-byte aligned", what);
  return WH_OK;
}

int launch_tree_attend(wh_ctx *ctx, const wh_tree *t, const void *q, const void *k, const void *v, size_t stride, int in16,
                       const uint32_t *kv, size_t kv_stride, int cols, void *o, int out16, int heads, int kv_heads, int hd) {
  if (int rc = tree_check(ctx, "tree attention", t)) return rc;
  if (!q || !kv || !o || !k != !v) return wh_fail(ctx, WH_EARG, "tree attention: q, the cache, o, and k with v are needed");
  if (heads <= 0 || heads > ATTEND_HEADS || kv_heads <= 0 || heads % kv_heads || hd <= 0 || hd > 128 || hd % 4 || cols <= 0 || cols > 1 << 24)
    return wh_fail(ctx, WH_EARG, "tree attention: bad shape (heads %d, key heads %d, head_dim %d, cols %d)", heads, kv_heads, hd,
                   cols);
  if (stride < (size_t)heads * hd || stride > (size_t)1 << 23)
    return wh_fail(ctx, WH_EARG, "tree attention: rows of %d queries %zu apart", heads * hd, stride);
  if (kv_stride && kv_stride < (size_t)cols * kv_heads * hd)
    return wh_fail(ctx, WH_EARG, "tree attention: caches of %zu words %zu apart", (size_t)cols * kv_heads * hd, kv_stride);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)kv | (uintptr_t)o) % 4 || (in16 && stride % 2))
    return wh_fail(ctx, WH_EARG, "tree attention: buffers and rows must be 4-byte aligned");
  AttendArgs a{q, k, v, stride, kv, kv_stride, o, t->n, t->count, t->mask, t->mask_stride, t->batch, t->rows, (t->rows + 31) / 32,
               cols, heads, kv_heads, hd, 1.0f / sqrtf((float)hd), 1, 1, 1, few_block(hd), NODES, nullptr, nullptr};
  const int rows = t->rows * (heads / kv_heads), tiles = (rows + 15) / 16;
  // Which kernel: up to 32 rows (16 of larger heads, for want of registers) attend_kernel, as it shares nothing (4
  // requests' 16 rows of 20 heads of 64 values over 448 keys 8.5 us, 12.4 by attend_rows_kernel; 32 rows 10.7 and 12.8).
  // More rows need the blocks shared.  attend_rows_kernel's workgroups have 4 wavefronts where that is all the rows there
  // are (4 requests' 60 f32 rows of 8 heads of 128 values over 28 k keys 98 us, 108 with 8; 16 requests' 20 over 448 16.7 and
  // 18.6; f16 rows and heads of 64 values within 4 % either way) and 8 otherwise (100 f16 rows of 128 values over 28 k keys
  // 114 us, 135 with 4).
  const int most = hd <= 64 ? 2 : 1;  // tiles of attend_kernel
  const int rt = tiles > most && hd >= 8 && cols >= 4 ? tiles <= 4 ? 4 : 8 : 0, qt = std::min(tiles, most);
  if (rt) a.block = a.node_block = rows_block(hd);
  const int blocks = (cols + a.block - 1) / a.block + (t->mask && k ? (t->rows + a.node_block - 1) / a.node_block : 0);
  a.row_blocks = (tiles + (rt ? rt : qt) - 1) / (rt ? rt : qt);
  const size_t units = (size_t)t->batch * kv_heads * a.row_blocks;
  const size_t cus = ctx->cus > 0 ? ctx->cus : 256;
  a.kw = rt ? 1 : std::min(WAVES, blocks);
  // A second launch joins the splits, so a cache that one workgroup gets through in 4 blocks a wavefront (8 of
  // attend_rows_kernel's) stays whole (1500 keys of 8 heads of 64 values for 4 requests 12.2 us, 13.6 in parts).  Of a
  // longer one each has at least half as many (4000 keys 14.9 us, 17.9 with as many), and there are as many as keep the
  // rounds of workgroups that the CUs hold at once short and full (1500 keys of 20 heads of 100 values for 5 requests
  // 22.3 us with 2 splits, 28.8 with 3, whose last round has 44 workgroups for 256 CUs; 4 requests' 300 nodes of 8 heads
  // over 28 k keys 239 us, 276 with one round's number rounded up).  All of this goes by the cache's size, since the lengths
  // are on the device: a long cache of which little is in use is planned as a full one and pays the second launch.
  const int least = (rt ? 4 : 2) * a.kw;
  if (blocks > 2 * least) {
    const size_t slots = cus * (rt ? 2 : 1);
    size_t best = SIZE_MAX;
    for (int x = 1; x <= std::min(SPLITS, (blocks + least - 1) / least); x++) {
      const size_t cost = (units * x + slots - 1) / slots * ((blocks + x - 1) / x + least);
      if (cost < best) best = cost, a.splits = x;
    }
  }
  const size_t nodes = (size_t)t->batch * t->rows;
  if ((size_t)t->batch * a.row_blocks > 65535 || units * a.splits >= (size_t)1 << 22 || nodes * heads >= (size_t)1 << 25)  // (a launch's limits)
    return wh_fail(ctx, WH_EARG, "tree attention: %d heads of %zu nodes in one call", heads, nodes);
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "tree attention: %s", hipGetErrorString(e));
  if (a.splits > 1) {
    const size_t part = (size_t)a.splits * nodes * heads;
    if (!(a.po = (float *)wh_scratch(ctx, part * (hd + 4) * sizeof(float)))) return WH_EOOM;
    a.pml = a.po + part * hd;
  }
  // Caches of more than the 256 MB that the chip keeps are read past it (4 requests' 4 rows over 28 k keys of 8 heads of 128
  // values: 85 us, 95 through it); smaller ones may be found there by the next step (4 requests' 13 rows over 1300 keys:
  // 11.6 us, 15.1 past it), which a large one of which little is in use goes without.  attend_rows_kernel gains nothing by it.
  const bool once = kv_stride && a.row_blocks == 1 && 4 * (size_t)t->batch * kv_heads * hd * cols > (size_t)256 << 20;
  return in16 ? out16 ? attend_t<_Float16, true>(ctx, a, qt, rt, once) : attend_t<_Float16, false>(ctx, a, qt, rt, once)
              : out16 ? attend_t<float, true>(ctx, a, qt, rt, once) : attend_t<float, false>(ctx, a, qt, rt, once);
}

int launch_tree_accept(wh_ctx *ctx, const wh_tree *t, const uint32_t *picks, const wh_kept *w, int cols, int32_t *path,
                       int32_t *kept, uint32_t *next, int32_t *n_out, uint32_t *history, int history_cols) {
  if (int rc = tree_check(ctx, "tree accept", t)) return rc;
  if (!t->tokens || !t->mask || !picks || !path || !kept || !next || !n_out || cols <= 0 || (history && history_cols <= 0))
    return wh_fail(ctx, WH_EARG, "tree accept: tokens, masks, picks, positions and the outputs are needed");
  if (((uintptr_t)picks | (uintptr_t)path | (uintptr_t)kept | (uintptr_t)next | (uintptr_t)n_out | (uintptr_t)history) % 4)
    return wh_fail(ctx, WH_EARG, "tree accept: the arrays must be 4-byte aligned");
  if (w) {
    if (!w->k || !w->v || !w->kv || w->layers <= 0 || w->layers > 65535 || w->d <= 0 || w->d % 2 || w->d > 1 << 24)
      return wh_fail(ctx, WH_EARG, "tree accept: bad rows or caches (layers %d, d %d)", w->layers, w->d);
    if (w->stride < (size_t)w->d || w->stride > (size_t)1 << 31 || (w->layers > 1 && w->layer_stride < w->stride))
      return wh_fail(ctx, WH_EARG, "tree accept: rows of %d values %zu apart, layers %zu", w->d, w->stride, w->layer_stride);
    const size_t cache = (size_t)cols * w->d;
    if ((t->batch > 1 && w->kv_stride < cache) || (w->layers > 1 && w->kv_layer_stride < cache))
      return wh_fail(ctx, WH_EARG, "tree accept: caches of %zu words %zu and %zu apart", cache, w->kv_stride, w->kv_layer_stride);
    if ((size_t)t->batch * ((w->d + 255) / 256) >= (size_t)1 << 24)  // (a launch's limit)
      return wh_fail(ctx, WH_EARG, "tree accept: %d sequences' rows of %d values in one call", t->batch, w->d);
    if (((uintptr_t)w->k | (uintptr_t)w->v | (uintptr_t)w->kv) % 4 || (w->in16 && (w->stride % 2 || w->layer_stride % 2)))
      return wh_fail(ctx, WH_EARG, "tree accept: buffers and rows must be 4-byte aligned");
  }
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "tree accept: %s", hipGetErrorString(e));
  const AcceptArgs a{t->n, t->count, t->tokens, t->mask, picks, t->mask_stride, t->rows, (t->rows + 31) / 32, cols,
                     path, kept, next, n_out, history, history_cols};
  const size_t nodes = (size_t)t->batch * t->rows, masks = t->mask_stride ? t->mask_stride * t->batch : (size_t)t->rows * a.words;
  // One launch, each of whose workgroups walks its sequence's tree for itself, unless an output lies in what they read (32
  // sequences' 9 of 61 nodes in 4 layers of 1280 values 10.4 us, 13.2 in two launches; 4 sequences' 9 of 1000 9.9 and 12.8).
  auto apart = [&](const void *y, size_t words) {
    const struct {
      const void *p;
      size_t words;
    } in[] = {{t->n, (size_t)t->batch}, {t->count, (size_t)t->batch}, {t->tokens, nodes}, {t->mask, masks}, {picks, nodes}};
    for (const auto &x : in)
      if (x.p && y && (uintptr_t)y < (uintptr_t)x.p + 4 * x.words && (uintptr_t)x.p < (uintptr_t)y + 4 * words) return false;
    return true;
  };
  const bool one = w && apart(path, nodes) && apart(kept, t->batch) && apart(next, t->batch) && apart(n_out, t->batch) &&
                   apart(history, (size_t)t->batch * history_cols);
  if (!one) {
    ProfScope prof(ctx, "tree_accept", 0.0, 16.0 * nodes);
    wh_launch(ctx, accept_kernel, t->batch, 256, 0, a);
    if (int rc = wh_launched(ctx, "tree accept")) return rc;
  }
  if (!w) return WH_OK;
  const int parts = (w->d + 255) / 256;
  const KeepArgs ka{w->k, w->v, w->stride, w->layer_stride, w->kv, w->kv_stride, w->kv_layer_stride, w->d, parts, one};
  const dim3 grid(t->batch * parts, w->layers);
  ProfScope prof(ctx, "tree_keep", 0.0, 0.0);
  if (w->in16) wh_launch(ctx, keep_kernel<_Float16>, grid, 256, 0, a, ka);
  else wh_launch(ctx, keep_kernel<float>, grid, 256, 0, a, ka);
  return wh_launched(ctx, "tree keep");
}
