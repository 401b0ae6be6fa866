// Attention of a step's rows over caches in pages (include/wavo_hip.h, wh_page_attend; pages.h for their layout).
#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "pages.h"
#include "rows.h"
#include "xlane.h"

namespace {

using namespace rows;
using namespace pages;

struct PageAttendArgs {
  const void *q, *k, *v;
  size_t stride;
  Pages pages;
  void *o;
  int out16;
  const int32_t *n, *count;
  const uint32_t *mask;
  size_t mask_stride;
  int batch, rows, words, heads;
  float scale;
  int kw, row_blocks, qt;  // qt: tiles of 16 rows of a block
  // even: how many workgroups share all the tiles of a key head evenly (0: each has a block of rows to itself), and the tiles that
  // one takes at least; their outputs, two parts each: unnormalized [part][row][hd] and (maximum, sum, factor of the
  // maximum's exponent, -) [part][row].
  int even, least;
  float *po, *pml;
};

constexpr int WAVES = 8;             // wavefronts of a workgroup, at most
constexpr float LOWEST = -1e30f;     // the maximum of a row that has seen nothing
constexpr int JOIN_LDS = 128 << 10;  // bytes in which wavefronts' results are joined

// Whether a compute unit holds two workgroups, of 128 registers a thread, or one of 256.  Where tiles are shared out, two do better
// while a tile, its queries and outputs fit (f16 rows of 96 over 4 bits, 32 sequences of 1000 to 8191: 37 us for 39 alone), and
// worse where they spill (f16 rows of 128 over 4 bits spill 18 registers: 60 us for 47 alone, with f32 outputs 25: 67 for 55; f32
// rows of 96 18: 51 for 46; f16 pages of heads of 128: 157 for 112).  Without shares a block's start and end are
// hidden by the other workgroup's, which is worth some spilled registers over 4 bits (64 sequences of 100 to 1500, 16 key heads: f16
// rows of 128 spill 4, 38 us for 41 alone; f32 rows of 96 4, 38 for 44).
constexpr bool two_of(int z, int qt, bool half_rows, bool q4, bool even) { return qt == 1 && z < (q4 ? 3 + half_rows + !even : 3); }

// What a block of rows costs a workgroup before its first tile and behind its last (its reads that wait for each other, the
// wavefronts' results joined), as tiles of its time.  One row a key head, 32 sequences of 1000 to 8191: 50, 44, 41 and 42 us
// with 0, 8, 24 and 48 (over f16 pages 112, 110, 112 and 117); 100 rows, 8 sequences of 1000 to 8000: 53, 50, 44 and 50 with 0, 8, 48
// and 96.
constexpr __host__ __device__ int start_of(int qt) { return qt == 1 ? 24 : 48; }

// A sequence's tiles: the cache's, then the nodes'.
struct Share {
  int n, count, cached, tiles;
};
__device__ __forceinline__ Share share_of(const PageAttendArgs &a, int n, int count) {
  Share s;
  s.n = min(max(n, 0), a.pages.room);
  s.count = min(max(count, 0), a.rows);
  s.cached = (s.n + TILE - 1) / TILE;
  s.tiles = s.cached + (a.mask && a.k ? (s.count + TILE - 1) / TILE : 0);
  return s;
}
__device__ __forceinline__ Share share_of(const PageAttendArgs &a, int b) { return share_of(a, a.n[b], a.count ? a.count[b] : a.rows); }

// All the tiles of a key head in a row: sequence by sequence, block of `rows` rows by block, each at least one.  (Every key
// head's are shared out alike, so that all of them are in the same pages at about the same time.)  64 sequences at a time are
// kept in LDS: their lengths and counts, and how many tiles they and those before them have.
struct EvenLds {
  int n[64], count[64];
  uint32_t sum[64];
};
struct Even {
  const PageAttendArgs &a;
  EvenLds &lds;
  int rows, b0;             // of the 64, the first
  uint32_t all, per, before;  // tiles; those of a workgroup; those before the 64
  __device__ __forceinline__ uint32_t load(int base) {  // (the tiles of the 64)
    const int lane = threadIdx.x & 63, b = base + lane;
    int n = 0, count = 0;
    if (b < a.batch) n = a.n[b], count = a.count ? a.count[b] : a.rows;
    const Share s = share_of(a, n, count);
    uint32_t sum = blocks_of(s) * tiles_of(s);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    if (threadIdx.x < 64) lds.n[lane] = n, lds.count[lane] = count, lds.sum[lane] = sum;
    return __builtin_amdgcn_readlane(sum, 63);
  }
  // A block's: as many besides its own as its start and end take the time of.
  __device__ __forceinline__ uint32_t tiles_of(const Share &s) const { return start_of(rows / 16) + max(s.tiles, 1); }
  __device__ __forceinline__ uint32_t blocks_of(const Share &s) const {
    return (s.count * (a.heads / a.pages.kv_heads) + rows - 1) / rows;
  }
  // (by every thread of a workgroup)
  __device__ __forceinline__ Even(const PageAttendArgs &a, EvenLds &lds, int rows) : a(a), lds(lds), rows(rows), b0(0), before(0) {
    all = load(0);
    if (a.batch > 64) {
      for (int base = 64; base < a.batch; base += 64) {
        __syncthreads();
        all += load(base);
      }
      __syncthreads();
      load(0);
    }
    __syncthreads();
    all = __builtin_amdgcn_readfirstlane(all);
    per = max((all + a.even - 1) / a.even, (uint32_t)a.least);
  }
  // The next 64 sequences.
  __device__ __forceinline__ void next() {
    before += __builtin_amdgcn_readfirstlane(lds.sum[63]), b0 += 64;
    __syncthreads();
    load(b0);
    __syncthreads();
  }
  // The sequence of the tile at `place` (< all, and not before the 64), and its first tile's place.
  __device__ __forceinline__ void find(uint32_t place, int &b, Share &s, uint32_t &first) {
    for (;; next()) {
      const uint32_t sum = lds.sum[threadIdx.x & 63];
      const uint64_t past = __ballot(before + sum > place);
      if (!past) continue;
      const int l = __builtin_ctzll(past);
      b = b0 + l, first = before + (l ? __builtin_amdgcn_readlane(sum, l - 1) : 0u);
      s = share_of(a, __builtin_amdgcn_readfirstlane(lds.n[l]), __builtin_amdgcn_readfirstlane(lds.count[l]));
      return;
    }
  }
};

// A tile's share of a lane: words of K and V, and for 4 bits the factors of the positions of its scores and weights.
template <int Z, bool Q4>
struct Tile;
template <int Z>
struct Tile<Z, true> {
  uint32_t k[2 * Z], v[2 * Z];
  half8 kd[Z], vd[Z];
  static __device__ __forceinline__ void words(uint32_t (&w)[2 * Z], const uint32_t *p, int lane) {
    constexpr int T = 2 * Z, whole = T & ~3;
#pragma unroll
    for (int t = 0; t < whole; t += 4) {
      const u32x4 x = *(const u32x4 *)(p + t * 64 + lane * 4);
      w[t] = x[0], w[t + 1] = x[1], w[t + 2] = x[2], w[t + 3] = x[3];
    }
    if constexpr (T > whole) {
      const u32x2 x = *(const u32x2 *)(p + whole * 64 + lane * 2);
      w[whole] = x[0], w[whole + 1] = x[1];
    }
  }
  __device__ __forceinline__ void load_k(const uint32_t *p, int lane, int g) {
    words(k, p, lane);
#pragma unroll
    for (int c = 0; c < Z; c++) kd[c] = *(const half8 *)(p + 128 * Z + (g * Z + c) * 4);
  }
  __device__ __forceinline__ void load_v(const uint32_t *p, int lane, int g) {
    words(v, p + 144 * Z, lane);
#pragma unroll
    for (int c = 0; c < Z; c++) vd[c] = *(const half8 *)(p + 272 * Z + (g * Z + c) * 4);
  }
  // nibble - 8 of the 8 elements, exactly: nibbles are the last bits of 1024 + x and of 64 + x.  (The constants from registers, so
  // that a mask and its sum are one instruction.)
  uint32_t low = 0x000f000fu, high = 0x00f000f0u, large = 0x64006400u, small = 0x54005400u;
  __device__ __forceinline__ Tile() { asm volatile("" : "+s"(low), "+s"(high), "+v"(large), "+v"(small)); }
  __device__ __forceinline__ half8 open(uint32_t w) const {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 2; i++, w >>= 8) {
      const half2 x = __builtin_bit_cast(half2, (w & low) | large) - half2{(_Float16)1032, (_Float16)1032};
      const half2 y = __builtin_bit_cast(half2, (w & high) | small) - half2{(_Float16)72, (_Float16)72};
      r[2 * i] = __builtin_bit_cast(uint32_t, x), r[2 * i + 1] = __builtin_bit_cast(uint32_t, y);
    }
    return __builtin_bit_cast(half8, r);
  }
  // What stands in positions that are not there must not meet their zero weights.
  __device__ __forceinline__ void clear_v(uint32_t there) {
#pragma unroll
    for (int c = 0; c < Z; c++)
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (!(there >> e & 1)) vd[c][e] = (_Float16)0;
  }
};
template <int Z>
struct Tile<Z, false> {
  u32x4 k[2 * Z], v[2 * Z];
  __device__ __forceinline__ void load_k(const uint32_t *p, int lane, int) {
#pragma unroll
    for (int t = 0; t < 2 * Z; t++) k[t] = *(const u32x4 *)(p + (t * 64 + lane) * 4);
  }
  __device__ __forceinline__ void load_v(const uint32_t *p, int lane, int) {
#pragma unroll
    for (int t = 0; t < 2 * Z; t++) v[t] = *(const u32x4 *)(p + 512 * Z + (t * 64 + lane) * 4);
  }
  __device__ __forceinline__ half8 open(u32x4 w) const { return __builtin_bit_cast(half8, w); }
  __device__ __forceinline__ void clear_v(uint32_t there) {
#pragma unroll
    for (int t = 0; t < 2 * Z; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) v[t][e] &= (there >> (2 * e) & 1 ? 0xffffu : 0u) | (there >> (2 * e + 1) & 1 ? 0xffff0000u : 0u);
  }
};

// A row of queries (of one that is not there: the last one's).
template <typename T, int Z>
__device__ __forceinline__ void load_rows(const PageAttendArgs &a, int b, int kh, int row, int g, float (&f)[Z][8]) {
  const int group = a.heads / a.pages.kv_heads, r = min(row, a.rows * group - 1);
  load_query<T, Z>((const T *)a.q + ((size_t)b * a.rows + node_of(r, group)) * a.stride + (size_t)(kh * group + head_of(r, group)) * 32 * Z, g, 32 * Z, f);
}

// A workgroup takes one key head of a sequence, 16 * QT of its rows (the heads / kv_heads query heads of a node are rows next
// to each other) and a run of its tiles, of which each of its kw wavefronts takes every kw-th.
//   Scores transposed, S^T = K Q^T: lane 16g + i holds row i's scores of positions position_of(g, e), e < 8.  For 4 bits the
//   products are those of nibble - 8, exact in f16, chunk by chunk of 32 values, and every chunk's sum is multiplied by its
//   position's factor in f32: K is taken as it stands.
//   Outputs transposed, O^T = V^T P^T, with V's factors in the weights (but for OPEN): a chunk's 32 values of V share one
//   factor, so the operand of P for that chunk is p * d.
// The next tile's K is asked for as soon as this one's scores are done, and its V after this one's outputs; its page two tiles
// ahead.
//
// Precision: f32 queries are scaled by a power of two per row and split into two f16 parts, as are the weights (p * d) for
// f32 outputs: two products each, with an error of 2^-22.  Weights are exp2(s - max + 10 - E): the second part is no
// subnormal, and E, zero until a factor of V reaches 2, keeps p * d within f16.  P16 (f16 outputs): p is rounded to f16,
// off by 2^-11 of itself, beside the output's own rounding; the weights' sum stays f32.
//
// OPEN (4 bits and P16): V is multiplied by its factors as it is opened, once for all rows, and rounded to f16 (2^-11 of itself, as
// an f16 cache would hold it), so that weights are operands as they stand.  K is not: so opened it took 142 us for the 162 of
// the 100 rows below, and made the outputs' error against 64 bits 4e-4 for 2.6e-4 (of which their own rounding is 2.1e-4).
//
// What bounds it.  16 rows over f16 pages: HBM (64 sequences of 4000 positions, 8 key heads of 128: 179 us, 5.9 TB/s).  16 rows
// over 4 bits, a quarter of the bytes: the vector instructions that open them (60 % of the time), beside the starts and ends of blocks
// (32 sequences of 1000 to 8191: 41 us and 4 for the join, 3.7 TB/s).  More rows: vector instructions, 365 for 48 rows of 32
// positions, of which some 180 open nibbles: 74% of the time, and matrix instructions 28% (100 rows over 8 caches of 24 to 33 k
// positions, 8 key heads of 128: 148 us and 5 for the join, 460 TFLOP/s, some 40 more on a card that comes from idling).
//
// attend_part: the tiles from start to end of sequence b's block of rows from r0 on of a key head; into the outputs, or as part `part`.
template <int Z, int QT, int QP, bool P16, bool Q4>
__device__ __forceinline__ void attend_part(const PageAttendArgs &a, uint8_t *smem, int b, int kh, int r0, const Share &s, int start, int end, int part,
                                            float (&f)[Z][8]) {
  typedef typename std::conditional<QP == 2, float, _Float16>::type T;
  constexpr int hd = 32 * Z;
  constexpr bool SHARED = QT > 1, OPEN = Q4 && P16;  // SHARED: queries in LDS
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // (nothing that follows from it is kept in registers from one run to the next)
  const int lane = tid & 63, ki = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, m = lane & 15;
  const int group = a.heads / a.pages.kv_heads, total = s.count * group;
  const size_t row0 = (size_t)b * a.rows;
  end = min(end, s.tiles);
  const int cached = min(end, s.cached), slot = a.pages.shift - 5;
  // (nothing writes the table meanwhile: its numbers by scalar loads)
  typedef const __attribute__((address_space(4))) int32_t *Table;
  const Table table = (Table)(uintptr_t)(a.pages.table + (size_t)b * a.pages.table_stride);

  // The tiles that are there, in turn: `blk` is worked on, `next` is asked for, and the page of `after` is.
  auto id_of = [&](int tile) { return table[min(tile, cached - 1) >> slot]; };
  auto skip = [&](int &tile, int &id) {
    while (tile < cached && (uint32_t)id >= (uint32_t)a.pages.pages) tile += a.kw, id = id_of(tile);
  };
  auto at = [&](int tile, int id) {
    return (const uint32_t *)a.pages.pool + (size_t)id * a.pages.page_words + (size_t)((kh << slot) + (tile & ((1 << slot) - 1))) * tile_words(Q4, hd);
  };
  Tile<Z, Q4> w;
  int blk = start + ki, next = cached, next_id = -1;
  if (blk < cached) {
    int id = id_of(blk);
    skip(blk, id);
    if (blk < cached) {
      const uint32_t *p = at(blk, id);
      w.load_k(p, lane, g);
      __builtin_amdgcn_sched_barrier(0);  // (K first, as in the loop: waits count the loads in between)
      w.load_v(p, lane, g);
      __builtin_amdgcn_sched_barrier(0);
      next = blk + a.kw, next_id = id_of(next);
    }
  }

  half8 q[SHARED ? 1 : Z][QP];
  half8 *const qs = (half8 *)smem;                    // [t][c][part][lane]
  float *const cfs = (float *)(qs + QT * Z * QP * 64);  // [t][row]
  floatx4 acc[QT][2 * Z];
  float mx[QT], sum[QT], cf[QP == 2 ? QT : 1], digits = 10.0f;
  auto factor = [&](int t) { return cf[QP == 2 ? t : 0]; };
  bool far = false;  // whether a maximum is past FAR
  // (rows that are not there: zeros, whose scores disturb nobody)
  auto taken = [&](int row, half8 (&x)[Z][QP]) {
#pragma unroll
    for (int c = 0; c < Z; c++)
#pragma unroll
      for (int e = 0; e < 8; e++) f[c][e] = row < total ? f[c][e] : 0.0f;
    return split_query(f, a.scale, x);
  };
  if constexpr (SHARED) {
    for (int t = ki; t < QT; t += a.kw) {
      half8 x[Z][QP];
      load_rows<T, Z>(a, b, kh, r0 + 16 * t + m, g, f);
      const float y = taken(r0 + 16 * t + m, x);
      if (g == 0) cfs[16 * t + m] = y;
#pragma unroll
      for (int c = 0; c < Z; c++)
#pragma unroll
        for (int part = 0; part < QP; part++) qs[((t * Z + c) * QP + part) * 64 + lane] = x[c][part];
    }
    meet();
    if constexpr (QP == 2)
#pragma unroll
      for (int t = 0; t < QT; t++) cf[t] = cfs[16 * t + m];
  } else {
    cf[0] = taken(r0 + m, q);
  }
  if constexpr (QP == 1) cf[0] = a.scale * 1.44269504088896341f;
#pragma unroll
  for (int t = 0; t < QT; t++) {
    mx[t] = LOWEST, sum[t] = 0.0f;
#pragma unroll
    for (int x = 0; x < 2 * Z; x++) acc[t][x] = floatx4{};
  }
  int mine = lane;
  asm volatile("" : "+v"(mine));  // (one address and its offsets: not others made of it that take registers)
  auto query_of = [&](int t, int c, int part) {
    if constexpr (SHARED) return qs[mine + ((t * Z + c) * QP + part) * 64];
    else return q[c][part];
  };

  typedef float floatx8 __attribute__((ext_vector_type(8)));
  typedef typename std::conditional<P16, half8, floatx8>::type P;
  // Scores st of a tile into weights p: exp2 against the running maxima, and their sums.  seen(t): the lane's positions.  All of
  // the block's rows together, so that a branch parts them only once.
  auto weights = [&](floatx4 (&st)[QT][2], bool masked, auto seen, P (&p)[QT]) {
    if (masked)
#pragma unroll
      for (int t = 0; t < QT; t++) {
        const uint32_t s = seen(t);
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (!(s >> e & 1)) st[t][e >> 2][e & 3] = -INFINITY;
      }
    float top[QT], by[QT];
    bool past = false;
#pragma unroll
    for (int t = 0; t < QT; t++) {
      top[t] = st[t][0][0];
#pragma unroll
      for (int e = 1; e < 8; e++) top[t] = fmaxf(top[t], st[t][e >> 2][e & 3]);
      by[t] = fminf(fmaf(-mx[t], factor(t), digits), -LOWEST);
      past |= fmaf(top[t], factor(t), by[t]) > digits + SLACK;
    }
    // A maximum is moved, for all of a row's lanes, where one of them has a score well past it: otherwise they need not meet.
    if (far || __any(past)) {
#pragma unroll
      for (int t = 0; t < QT; t++) {
        const float c = factor(t);
        if (!__any(fmaf(top[t] - mx[t], c, digits) > digits + SLACK)) continue;
        top[t] = xlane::bit4(top[t], xlane::Max{});
        top[t] = fmaxf(xlane::bit5(top[t], xlane::Max{}), mx[t]);
        const float old = __builtin_amdgcn_exp2f((mx[t] - top[t]) * c);
        sum[t] *= old;
#pragma unroll
        for (int x = 0; x < 2 * Z; x++) acc[t][x] *= old;
        mx[t] = top[t];
        by[t] = fminf(fmaf(-top[t], c, digits), -LOWEST);
        far = far || __any(top[t] != LOWEST && fabsf(by[t]) > FAR);
      }
      if (far)
#pragma unroll
        for (int t = 0; t < QT; t++) st[t][0] -= mx[t], st[t][1] -= mx[t], by[t] = digits;
    }
#pragma unroll
    for (int t = 0; t < QT; t++)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(st[t][e >> 2][e & 3], factor(t), by[t]));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(st[t][e >> 2][e + 1 & 3], factor(t), by[t]));
        sum[t] += p0, sum[t] += p1;
        if constexpr (P16) weights2<true>(p0, p1, p[t], p[t], e);
        else p[t][e] = p0, p[t][e + 1] = p1;
      }
  };
  // p times a chunk's factors as an operand, and (unless P16) what that leaves of them.
  auto operand = [&](const P &p, const half8 *d, half8 &h, half8 &l) {
    if constexpr (P16) {
      h = d ? p * *d : p;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        weights2<false>(d ? p[e] * (float)(*d)[e] : p[e], d ? p[e + 1] * (float)(*d)[e + 1] : p[e + 1], h, l, e);
    }
  };
  // Factors of V of 2 and more: the weights that follow are smaller by their largest's power of two.
  auto room = [&] {
    if constexpr (Q4 && !OPEN) {
      uint32_t any = 0;
#pragma unroll
      for (int c = 0; c < Z; c++) {
        const u32x4 x = __builtin_bit_cast(u32x4, w.vd[c]);
        any |= x[0] | x[1] | x[2] | x[3];
      }
      if (__any(any & 0x40004000u)) {
        float most = 0.0f;
#pragma unroll
        for (int c = 0; c < Z; c++)
#pragma unroll
          for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf((float)w.vd[c][e]));
        most = xlane::wave_max(most);
        const float want = 10.0f - fminf((float)(__builtin_amdgcn_frexp_expf(most) - 1), 15.0f);  // (most < 2^(10 - want + 1))
        if (most >= 2.0f && want < digits) {
          const float less = __builtin_amdgcn_exp2f(want - digits);
#pragma unroll
          for (int t = 0; t < QT; t++) {
            sum[t] *= less;
#pragma unroll
            for (int x = 0; x < 2 * Z; x++) acc[t][x] *= less;
          }
          digits = want;
        }
      }
    }
  };

  auto step = [&](auto more) {
    int after = next + a.kw, after_id = 0;
    if constexpr (more) after_id = id_of(after);
    const uint32_t *np = at(next, next_id);
    floatx4 st[QT][2];
#pragma unroll
    for (int t = 0; t < QT; t++) st[t][0] = st[t][1] = floatx4{};
    // (matrix instructions of a word among the vector ones that open the next)
    // (and queries asked for when the chunk before them is done)
    half8 k = w.open(w.k[0]), x[QT][QP];
#pragma unroll
    for (int t = 0; t < QT; t++)
#pragma unroll
      for (int part = 0; part < QP; part++) x[t][part] = query_of(t, 0, part);
    if constexpr (QT > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2 * Z; i++) {
      const int c = i / 2, u = i % 2;
      half8 after = k;
      floatx4 y[QT];
      if (i + 1 < 2 * Z) after = w.open(w.k[i + 1]);
#pragma unroll
      for (int t = 0; t < QT; t++) {
        if constexpr (Q4) {
          y[t] = mfma(k, x[t][0], floatx4{});
          if constexpr (QP == 2) y[t] = mfma(k, x[t][QP - 1], y[t]);
        } else {
#pragma unroll
          for (int part = 0; part < QP; part++) st[t][u] = mfma(k, x[t][part], st[t][u]);
        }
        if (u == 1 && c + 1 < Z)
#pragma unroll
          for (int part = 0; part < QP; part++) x[t][part] = query_of(t, c + 1, part);
      }
      if constexpr (Q4)
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) st[t][u][r] = fmaf(y[t][r], (float)w.kd[c][4 * u + r], st[t][u][r]);
      k = after;
      if constexpr (QT > 1 && OPEN) {
#pragma unroll
        for (int t = 0; t < QT; t++) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (u == 1 && c + 1 < Z) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, (9 + QT - 1) / QT, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // (the scores are done before K's registers take the next tile: it would be waited for at the end of this one otherwise)
#pragma unroll
    for (int t = 0; t < QT; t++) asm volatile("" : "+v"(st[t][0]), "+v"(st[t][1]));
    if constexpr (more) w.load_k(np, lane, g);
    const int left = s.n - TILE * blk;
    uint32_t seen = 0xff;
    if (left < TILE) {
      const uint32_t there = (1u << left) - 1u;
      seen = (there >> 4 * g & 15) | (there >> (16 + 4 * g) & 15) << 4;
      w.clear_v(seen);
    }
    room();
    P p[QT];
    weights(st, left < TILE, [&](int) { return seen; }, p);
    auto open_v = [&](int i) {
      half8 v = w.open(w.v[i]);
      if constexpr (OPEN) v *= w.vd[i / 2];
      return v;
    };
    half8 v = open_v(0);
    if constexpr (QT > 1) __builtin_amdgcn_sched_barrier(0);
    half8 h[QT], l[QT];
#pragma unroll
    for (int i = 0; i < 2 * Z; i++) {
      half8 after = v;
      if (i + 1 < 2 * Z) after = open_v(i + 1);
#pragma unroll
      for (int t = 0; t < QT; t++) {
        if (i % 2 == 0) {
          if constexpr (Q4 && !OPEN) operand(p[t], &w.vd[i / 2], h[t], l[t]);
          else operand(p[t], nullptr, h[t], l[t]);
        }
        acc[t][i] = mfma(v, h[t], acc[t][i]);
        if constexpr (!P16) acc[t][i] = mfma(v, l[t], acc[t][i]);
      }
      v = after;
      if constexpr (QT > 1 && OPEN) {
#pragma unroll
        for (int t = 0; t < QT; t++) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, (13 + QT - 1) / QT, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (more) {
      w.load_v(np, lane, g);
      blk = next, next = after, next_id = after_id;
    }
  };
  if (blk < cached) {
    for (skip(next, next_id); next < cached; skip(next, next_id)) step(std::true_type{});
    step(std::false_type{});
  }

  // The nodes, 32 at a time: K and V as f16.
  const int first = max(start, s.cached);
  const uint32_t *masks = a.mask ? a.mask + (size_t)b * a.mask_stride : nullptr;
  auto mask_of = [&](int t, int word) { return masks[(size_t)node_of(min(r0 + 16 * t + m, a.rows * group - 1), group) * a.words + word]; };
  for (int tile = first + ((ki - (first - start)) % a.kw + a.kw) % a.kw; tile < end; tile += a.kw) {
    const int j0 = TILE * (tile - s.cached), last = s.count - 1 - j0;
    const T *k = (const T *)a.k + (row0 + j0) * a.stride + (size_t)kh * hd, *v = (const T *)a.v + (row0 + j0) * a.stride + (size_t)kh * hd;
    const uint32_t there = last >= TILE - 1 ? 0xffffffffu : (2u << last) - 1u;
    floatx4 st[QT][2];
#pragma unroll
    for (int t = 0; t < QT; t++) st[t][0] = st[t][1] = floatx4{};
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const T *row = k + (size_t)min(16 * u + m, last) * a.stride + 8 * g;
      typename Four<T>::type raw[Z][2];
#pragma unroll
      for (int c = 0; c < Z; c++) raw[c][0] = raw4(row + 32 * c), raw[c][1] = raw4(row + 32 * c + 4);
#pragma unroll
      for (int c = 0; c < Z; c++) {
        const u32x2 x = pairs4(raw[c][0]), y = pairs4(raw[c][1]);
        const half8 kf = __builtin_bit_cast(half8, u32x4{x[0], x[1], y[0], y[1]});
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int part = 0; part < QP; part++) st[t][u] = mfma(kf, query_of(t, c, part), st[t][u]);
      }
    }
    P p[QT];
    weights(st, true, [&](int t) {
      const uint32_t sees = there & mask_of(t, j0 / 32);
      return (sees >> 4 * g & 15) | (sees >> (16 + 4 * g) & 15) << 4;
    }, p);
#pragma unroll
    for (int c = 0; c < Z; c++) {
      // Values of nodes that are not there are zeroed, and so are those that are no finite numbers: they must not meet the zero
      // weights of the rows that do not see them, and are added to the others' outputs one by one.
      uint32_t x[8];
      u16x2 big{};
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const T *y = v + (size_t)min(position_of(g, e), last) * a.stride + 32 * c + 2 * m;
        if constexpr (QP == 2) {
          typedef floatx2 any __attribute__((aligned(4)));
          const floatx2 f2 = *(const any *)y;
          x[e] = pack2(f2[0], f2[1]);
        } else {
          x[e] = *(const uint32_t *)y;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (position_of(g, e) > last) x[e] = 0;
        big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, x[e] & 0x7fff7fffu));
      }
      if (__any(big[0] >= 0x7c00 || big[1] >= 0x7c00)) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = finite2(x[e]);
#pragma unroll 1
        for (int j = 0; j < min(TILE, last + 1); j++) {
          const T *y = v + (size_t)j * a.stride;
#pragma unroll
          for (int t = 0; t < QT; t++) {
            if (!(mask_of(t, j0 / 32) >> j & 1)) continue;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
              for (int r = 0; r < 4; r++) acc[t][2 * c + i][r] += not_finite(y, 32 * c + 8 * g + 2 * r + i, hd);
          }
        }
      }
      u32x4 v0, v1;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        v0[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);
        v1[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);
      }
#pragma unroll
      for (int t = 0; t < QT; t++) {
        half8 h, l;
        operand(p[t], nullptr, h, l);
        const half8 a0 = __builtin_bit_cast(half8, v0), a1 = __builtin_bit_cast(half8, v1);
        acc[t][2 * c] = mfma(a0, h, acc[t][2 * c]), acc[t][2 * c + 1] = mfma(a1, h, acc[t][2 * c + 1]);
        if constexpr (!P16) acc[t][2 * c] = mfma(a0, l, acc[t][2 * c]), acc[t][2 * c + 1] = mfma(a1, l, acc[t][2 * c + 1]);
      }
    }
  }

  // The wavefronts' results joined through LDS, where the queries were: half of them added to the other half until the rest fit,
  // which write their own, and every lane adds up four values of a row.  Lane 16g + i holds row i's values 32c + 8g + 2r + x.
  constexpr int SLOT = QT * Z * 128, FIT = JOIN_LDS / (16 * SLOT);
  const float more = __builtin_amdgcn_exp2f(10.0f - digits);
#pragma unroll
  for (int t = 0; t < QT; t++) {
    sum[t] = xlane::bit4(sum[t], xlane::Add{});
    sum[t] = xlane::bit5(sum[t], xlane::Add{}) * more;
    if constexpr (Q4 && !OPEN)
#pragma unroll
      for (int x = 0; x < 2 * Z; x++) acc[t][x] *= more;
  }
  int waves = a.kw;
  floatx4 *merge = (floatx4 *)smem;                             // [wave][...][lane]
  float *ml = (float *)(merge + min(waves, FIT) * SLOT);  // [wave][t][maxima, sums][row]
  if constexpr (SHARED) meet();
  if constexpr (FIT < WAVES)
    for (; waves > FIT; waves /= 2) {
      const int half = waves / 2;
      if (ki >= half && ki < waves) {
#pragma unroll
        for (int t = 0; t < QT; t++) {
          if (g == 0) ml[32 * ((ki - half) * QT + t) + m] = mx[t], ml[32 * ((ki - half) * QT + t) + 16 + m] = sum[t];
#pragma unroll
          for (int x = 0; x < 2 * Z; x++) merge[(ki - half) * SLOT + (t * 2 * Z + x) * 64 + lane] = acc[t][x];
        }
      }
      meet();
      if (ki < half) {
#pragma unroll
        for (int t = 0; t < QT; t++) {
          const float om = ml[32 * (ki * QT + t) + m], os = ml[32 * (ki * QT + t) + 16 + m], top = fmaxf(mx[t], om);
          const float y = mx[t] == top ? 1.0f : __builtin_amdgcn_exp2f((mx[t] - top) * factor(t)), z = om == top ? 1.0f : __builtin_amdgcn_exp2f((om - top) * factor(t));
          mx[t] = top, sum[t] = sum[t] * y + os * z;
#pragma unroll
          for (int x = 0; x < 2 * Z; x++) acc[t][x] = acc[t][x] * y + merge[ki * SLOT + (t * 2 * Z + x) * 64 + lane] * z;
        }
      }
      meet();
    }
  if (ki < waves) {
#pragma unroll
    for (int t = 0; t < QT; t++) {
      if (g == 0) ml[32 * (ki * QT + t) + m] = mx[t], ml[32 * (ki * QT + t) + 16 + m] = sum[t];
#pragma unroll
      for (int c = 0; c < Z; c++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          merge[ki * SLOT + ((t * Z + c) * 2 + h) * 64 + lane] =
              floatx4{acc[t][2 * c][2 * h], acc[t][2 * c + 1][2 * h], acc[t][2 * c][2 * h + 1], acc[t][2 * c + 1][2 * h + 1]};
    }
  }
  meet();
  for (int x = ki; x < QT * Z * 2; x += a.kw) {
    const int t = x / (2 * Z), c = x / 2 % Z, d = 32 * c + 8 * g + 4 * (x % 2), r = r0 + 16 * t + m;
    if (r >= total) continue;
    constexpr int MOST = std::min(WAVES, FIT);
    float km[MOST], kl[MOST], top = -INFINITY, l = 0.0f, scale = cf[0];
    if constexpr (QP == 2)
#pragma unroll
      for (int y = 1; y < QT; y++) scale = t == y ? cf[y] : scale;
    floatx4 kf[MOST], o{};
#pragma unroll
    for (int k = 0; k < MOST; k++) {
      const int y = min(k, waves - 1);
      km[k] = ml[32 * (y * QT + t) + m], kl[k] = ml[32 * (y * QT + t) + 16 + m], kf[k] = merge[y * SLOT + x * 64 + lane];
      if (k >= waves) km[k] = -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < MOST; k++) top = fmaxf(top, km[k]);
#pragma unroll
    for (int k = 0; k < MOST; k++) {
      if (k >= waves) break;
      const float y = km[k] == top ? 1.0f : __builtin_amdgcn_exp2f((km[k] - top) * scale);
      l += y * kl[k], o += y * kf[k];
    }
    const int i = node_of(r, group), head = kh * group + head_of(r, group);
    const size_t out = ((row0 + i) * a.heads + head) * hd + d;
    if (part >= 0) {
      const size_t row = (size_t)part * 16 * QT + 16 * t + m;
      if (d == 0) *(floatx4 *)(a.pml + 4 * row) = floatx4{top, l, scale, 0.0f};
      *(floatx4 *)(a.po + row * hd + d) = o;
      continue;
    }
    o *= l == 0.0f ? 0.0f : 1.0f / l;
    if (a.out16) *(u32x2_a4 *)((_Float16 *)a.o + out) = u32x2{pack2(o[0], o[1]), pack2(o[2], o[3])};
    else *(floatx4_a4 *)((float *)a.o + out) = o;
  }
}

// EVEN: the workgroups take runs of all the tiles, of the same length, whatever sequences' they are.
template <int Z, int QT, int QP, bool P16, bool Q4, bool EVEN>
__global__ __launch_bounds__(64 * WAVES, two_of(Z, QT, QP == 1, Q4, EVEN) ? 4 : 2) void page_attend_kernel(PageAttendArgs a) {
  typedef typename std::conditional<QP == 2, float, _Float16>::type T;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int g = threadIdx.x >> 4 & 3, m = threadIdx.x & 15, group = a.heads / a.pages.kv_heads;
  float f[Z][8];
  if constexpr (EVEN) {
    __shared__ EvenLds lds;
    Even even(a, lds, 16 * QT);
    const uint32_t last = min((blockIdx.y + 1) * even.per, even.all);
    const int kh = blockIdx.x;
    for (uint32_t place = blockIdx.y * even.per; place < last;) {
      int b;
      Share s;
      uint32_t first;
      even.find(place, b, s, first);
      const uint32_t tiles = even.tiles_of(s), block = (place - first) / tiles;
      first += block * tiles;
      const int r0 = 16 * QT * block, start = max((int)(place - first) - start_of(QT), 0), end = (int)min(tiles, last - first) - start_of(QT);
      place = first + tiles;
      if (end <= start) continue;
      if constexpr (QT == 1) load_rows<T, Z>(a, b, kh, r0 + m, g, f);
      attend_part<Z, QT, QP, P16, Q4>(a, smem, b, kh, r0, s, start, end, start || place > last ? (int)(2 * (kh * a.even + blockIdx.y) + !start) : -1, f);
      if (place < last) meet();
    }
  } else {
    const int kh = blockIdx.x, b = a.row_blocks == 1 ? blockIdx.y : blockIdx.y / a.row_blocks, r0 = 16 * QT * (blockIdx.y - b * a.row_blocks);
    if constexpr (QT == 1) load_rows<T, Z>(a, b, kh, r0 + m, g, f);  // (nothing is known of the lengths yet)
    const Share s = share_of(a, b);
    if constexpr (QT == 1)  // (asked for above, with the lengths, and not where they are first used)
#pragma unroll
      for (int c = 0; c < Z; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) asm volatile("" : "+v"(f[c][e]));
    if (r0 < s.count * group) attend_part<Z, QT, QP, P16, Q4>(a, smem, b, kh, r0, s, 0, s.tiles, -1, f);
  }
}

// The parts of a block of rows joined, where it has several: 8 rows a workgroup, four values a thread.
__global__ __launch_bounds__(256) void page_join_kernel(PageAttendArgs a) {
  __shared__ EvenLds lds;
  const int hd = a.pages.hd, group = a.heads / a.pages.kv_heads, rows = 16 * a.qt;
  Even even(a, lds, rows);
  const int unit = blockIdx.x, rb = unit % a.row_blocks, kh = unit / a.row_blocks % a.pages.kv_heads, b = unit / a.row_blocks / a.pages.kv_heads;
  while (b >= even.b0 + 64) even.next();
  const Share s = share_of(a, lds.n[b - even.b0], lds.count[b - even.b0]);
  const int blocks = even.blocks_of(s), local = 8 * blockIdx.y + threadIdx.x / 32, d = 4 * (threadIdx.x % 32), r = rows * rb + local;
  if (rb >= blocks || r >= s.count * group || d >= hd) return;
  const uint32_t tiles = even.tiles_of(s), first = even.before + (b > even.b0 ? lds.sum[b - even.b0 - 1] : 0u) + (uint32_t)rb * tiles;
  const int w0 = (first + start_of(a.qt)) / even.per, w1 = (first + tiles - 1) / even.per;
  if (w0 == w1) return;
  auto at = [&](int w) { return (size_t)(2 * (kh * a.even + w) + (w == w0)) * rows + local; };
  float top = -INFINITY, l = 0.0f;
  floatx4 o{};
  for (int w = w0; w <= w1; w += 4) {
    // (four parts at a time; those past the last: the last, not counted)
    floatx4 y[4], x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = *(const floatx4 *)(a.pml + 4 * at(min(w + i, w1))), x[i] = *(const floatx4 *)(a.po + at(min(w + i, w1)) * hd + d);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (w + i > w1) break;
      const float more = fmaxf(top, y[i][0]), u = top == more ? 1.0f : __builtin_amdgcn_exp2f((top - more) * y[i][2]);
      const float v = y[i][0] == more ? 1.0f : __builtin_amdgcn_exp2f((y[i][0] - more) * y[i][2]);
      l = l * u + y[i][1] * v, o = o * u + x[i] * v, top = more;
    }
  }
  o *= l == 0.0f ? 0.0f : 1.0f / l;
  const size_t out = (((size_t)b * a.rows + node_of(r, group)) * a.heads + kh * group + head_of(r, group)) * hd + d;
  if (a.out16) *(u32x2_a4 *)((_Float16 *)a.o + out) = u32x2{pack2(o[0], o[1]), pack2(o[2], o[3])};
  else *(floatx4_a4 *)((float *)a.o + out) = o;
}

template <int Z, int QT, int QP, bool P16, bool Q4>
int attend_launch(wh_ctx *ctx, const PageAttendArgs &a) {
  const double keys = (double)a.batch * a.pages.room;
  ProfScope prof(ctx, "page_attend", 4.0 * keys * a.rows * a.heads * a.pages.hd, keys * a.pages.kv_heads * a.pages.hd * (Q4 ? 1.125 : 4.0));
  const size_t join = (size_t)std::min(a.kw, JOIN_LDS / (QT * Z * 2048)) * QT * (Z * 2048 + 128), queries = QT > 1 ? QT * (Z * QP * 1024 + 64) : 0;
  const size_t shm = std::max(join, queries);
  if (a.even) wh_launch(ctx, (page_attend_kernel<Z, QT, QP, P16, Q4, true>), dim3(a.pages.kv_heads, a.even), 64 * a.kw, shm, a);
  else wh_launch(ctx, (page_attend_kernel<Z, QT, QP, P16, Q4, false>), dim3(a.pages.kv_heads, a.batch * a.row_blocks), 64 * a.kw, shm, a);
  return wh_launched(ctx, "page attention");
}
template <int Z, int QP, bool P16, bool Q4>
int attend_qt(wh_ctx *ctx, const PageAttendArgs &a, int qt) {
  if constexpr (P16) {
    if (qt == 3) return attend_launch<Z, 3, QP, P16, Q4>(ctx, a);
  }
  return qt == 1 ? attend_launch<Z, 1, QP, P16, Q4>(ctx, a) : attend_launch<Z, 2, QP, P16, Q4>(ctx, a);
}
template <int QP, bool P16, bool Q4>
int attend_z(wh_ctx *ctx, const PageAttendArgs &a, int qt) {
  switch (a.pages.hd / 32) {
    case 1: return attend_qt<1, QP, P16, Q4>(ctx, a, qt);
    case 2: return attend_qt<2, QP, P16, Q4>(ctx, a, qt);
    case 3: return attend_qt<3, QP, P16, Q4>(ctx, a, qt);
    default: return attend_qt<4, QP, P16, Q4>(ctx, a, qt);
  }
}
template <bool Q4>
int attend_types(wh_ctx *ctx, const PageAttendArgs &a, int in16, int out16, int qt) {
  return !in16 ? attend_z<2, false, Q4>(ctx, a, qt) : out16 ? attend_z<1, true, Q4>(ctx, a, qt) : attend_z<1, false, Q4>(ctx, a, qt);
}

}  // namespace

int launch_page_attend(wh_ctx *ctx, const wh_tree *t, const void *q, const void *k, const void *v, size_t stride, int in16, const wh_pages *p,
                       void *o, int out16, int heads) {
  if (int rc = tree_check(ctx, "page attention", t)) return rc;
  if (int rc = pages_check(ctx, "page attention", p)) return rc;
  if (!q || !o || !k != !v) return wh_fail(ctx, WH_EARG, "page attention: q, o, and k with v are needed");
  if (heads <= 0 || heads > ATTEND_HEADS || heads % p->kv_heads)
    return wh_fail(ctx, WH_EARG, "page attention: %d heads over %d of keys", heads, p->kv_heads);
  if (stride < (size_t)heads * p->hd || stride > (size_t)1 << 23)
    return wh_fail(ctx, WH_EARG, "page attention: rows of %d queries %zu apart", heads * p->hd, stride);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) % 4 || (in16 && stride % 2))
    return wh_fail(ctx, WH_EARG, "page attention: buffers and rows must be 4-byte aligned");
  PageAttendArgs a{q, k, v, stride, pages_of(p), o, out16 != 0, t->n, t->count, t->mask, t->mask_stride, t->batch, t->rows, (t->rows + 31) / 32,
                   heads, 1.0f / sqrtf((float)p->hd), 1, 1, 1, 0, 0, nullptr, nullptr};
  const int tiles = a.pages.room / TILE + (t->mask && k ? (t->rows + TILE - 1) / TILE : 0);
  while (2 * a.kw <= std::min(WAVES, tiles)) a.kw *= 2;
  const bool shared = tiles > 8 * a.kw;
  // Rows in tiles of 16, evenly in blocks of `most` at most.  3 tiles read a tile of the cache, and open its nibbles, once for 48
  // rows: with 32 query heads over 8 of 128 and f16 throughout, 100 rows over 28 k positions take 160 us for 165 with 2, 296 for 384
  // over f16 pages (heads of 64: 102 for 107, 147 for 189), over 5 k 47 for 46, and 58 for 63.  f16 pages that are not shared out do
  // better with more workgroups (8 times 48 rows over 200 to 1500, 8 key heads: 20 us for 16 with 2).  4 spill registers (192; 3 spill
  // 8 or 9 in heads of 128), and f32 weights and outputs leave registers for 2.
  const int rows = (t->rows * (heads / p->kv_heads) + 15) / 16, most = in16 && out16 && (shared || p->type == WH_Q4_0) ? 3 : 2;
  a.row_blocks = (rows + most - 1) / most;
  const int qt = (rows + a.row_blocks - 1) / a.row_blocks;
  a.row_blocks = (rows + qt - 1) / qt, a.qt = qt;
  const size_t blocks = (size_t)t->batch * a.row_blocks, units = blocks * p->kv_heads, nodes = (size_t)t->batch * t->rows;
  const size_t cus = ctx->cus > 0 ? ctx->cus : 256;
  if (shared && blocks * (tiles + start_of(qt)) < (size_t)1 << 31) {
    a.even = (int)std::max<size_t>(cus * (two_of(p->hd / 32, qt, in16, p->type == WH_Q4_0, true) ? 2 : 1) / p->kv_heads, 1);
    a.least = start_of(qt) + a.kw;
  }
  if (blocks > 65535 || units >= (size_t)1 << 22 || nodes * heads >= (size_t)1 << 25)  // (a launch's limits)
    return wh_fail(ctx, WH_EARG, "page attention: %d heads of %zu nodes in one call", heads, nodes);
  const size_t in = in16 ? 2 : 4, out = (size_t)heads * p->hd * (out16 ? 2 : 4);
  auto over = [&](const void *x, int of) { return x && rows_meet(o, out, out, x, (size_t)of * p->hd * in, stride * in, nodes); };
  if (over(q, heads) || over(k, p->kv_heads) || over(v, p->kv_heads)) return wh_fail(ctx, WH_EARG, "page attention: the output overlaps the rows");
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "page attention: %s", hipGetErrorString(e));
  if (a.even) {
    const size_t part_rows = (size_t)2 * a.even * p->kv_heads * 16 * qt;
    if (!(a.po = (float *)wh_scratch(ctx, part_rows * (p->hd + 4) * sizeof(float)))) return WH_EOOM;
    a.pml = a.po + part_rows * p->hd;
  }
  if (int rc = p->type == WH_Q4_0 ? attend_types<true>(ctx, a, in16, out16, qt) : attend_types<false>(ctx, a, in16, out16, qt)) return rc;
  if (!a.even) return WH_OK;
  ProfScope prof(ctx, "page_attend_join", 0.0, 8.0 * a.even * p->kv_heads * 16 * qt * (p->hd + 4));
  wh_launch(ctx, page_join_kernel, dim3((unsigned)units, 2 * qt), 256, 0, a);
  return wh_launched(ctx, "page attention's join");
}
