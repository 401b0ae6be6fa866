// Rows of a projection on their way into attention and into caches in pages (include/wavo_hip.h): norms of queries and
// keys per head with the rotation by their positions, and storing and reading keys and values of 4 or 16 bits.
#include <algorithm>

#include "internal.h"
#include "pages.h"
#include "rows.h"
#include "xlane.h"

namespace {

using namespace rows;
using namespace pages;

typedef _Float16 half4 __attribute__((ext_vector_type(4)));

// The norms and the rotation of a step's queries and keys.
struct Turn {
  const float *q_gain, *k_gain;
  float eps;
  const float *table;
  int positions, rot, pairs;
};

struct NormArgs {
  Turn turn;
  const void *x;
  size_t stride;
  void *y;
  size_t y_stride;
  const int32_t *n, *count;
  const uint32_t *mask;  // depths by the masks, where there are any; otherwise row by row
  size_t mask_stride;
  int rows, words, heads, turned, all, hd;  // heads: queries; turned: and keys; all: and values that are copied
  int per, in16, out16;                     // lanes of a head
};

__device__ __forceinline__ floatx4 load4(const void *x, size_t at, int in16) {
  floatx4 f;
  if (in16) values((const _Float16 *)x + at, (float *)&f);
  else f = raw4((const float *)x + at);
  return f;
}
__device__ __forceinline__ void store4(void *y, size_t at, int out16, floatx4 f) {
  if (out16) *(u32x2_a4 *)((_Float16 *)y + at) = pairs4(f);
  else *(floatx4_a4 *)((float *)y + at) = f;
}

// The sum over a head's lanes: per of them next to each other, a power of two, 32 at most.
__device__ __forceinline__ float head_sum(float v, int per) {
  if (per > 1) v += xlane::dpp<xlane::XOR1>(v);
  if (per > 2) v += xlane::dpp<xlane::XOR2>(v);
  if (per > 4) v += xlane::dpp<xlane::HALF_MIRROR>(v);
  if (per > 8) v += xlane::dpp<xlane::MIRROR>(v);
  if (per > 16) v = xlane::bit4(v, xlane::Add{});
  return v;
}

// How many nodes below i node i sees, which is its depth in a tree.
__device__ __forceinline__ int depth_of(const uint32_t *mask, int i) {
  int d = 0;
  for (int w = 0; w < i / 32; w++) d += __popc(mask[w]);
  return d + (i % 32 ? __popc(mask[i / 32] & ((1u << i % 32) - 1u)) : 0);
}

constexpr int NORM_THREADS = 256;

// A row's heads, `per` lanes each, by a workgroup: lane i holds 4 values of the head from `first` and 4 from `second` on, which
// the rotation turns against each other, so that a head is read and written once, in pieces of 8 or 16 bytes, and its squares meet
// in a few lane exchanges.  Bound by HBM: 8192 rows of 48 f16 heads of 128 take 42 us, 4.8 TB/s, f32 ones 78.  (One token: 4 us, a
// launch and three reads that wait for each other.)  H: f16 rows, whose squares never leave f32.  f32 rows' may, and the branch for
// those makes the next head's loads wait for this one's sums (100 us for 93 where 8192 rows are appended), so they are asked for first.
template <bool H>
__device__ __forceinline__ void norm_heads(const NormArgs &a, size_t row, int position, int tid, int threads) {
  const int per = a.per, at = tid / per, lane = tid % per, half = a.turn.rot / 2, hd = a.hd;
  const bool there = 8 * lane < hd;
  int first = 8 * lane, second = first + 4;  // neighbours
  bool turns = a.turn.table && first < a.turn.rot;
  if (turns && !a.turn.pairs) first = 4 * lane, second = first + half;
  if (!there) first = second = 0;
  float c[4], s[4];
  if (turns) {
    const float *t = a.turn.table + (size_t)min(max(position, 0), a.turn.positions - 1) * a.turn.rot;
    const int i = a.turn.pairs ? first / 2 : first;
#pragma unroll
    for (int e = 0; e < 4; e++) c[e] = t[i + e], s[e] = t[half + i + e];
  }
  auto load = [&](int head, floatx4 &u, floatx4 &w) {
    const size_t from = row * a.stride + (size_t)head * hd;
    u = load4(a.x, from + first, H), w = load4(a.x, from + second, H);
  };
  floatx4 next_u{}, next_w{};
  if (!H && at < a.all) load(at, next_u, next_w);
  for (int head = at, next; head < a.all; head = next) {
    next = head + threads / per;
    const size_t to = row * a.y_stride + (size_t)head * hd;
    floatx4 u = next_u, w = next_w;
    if (H) load(head, u, w);
    else if (next < a.all) load(next, next_u, next_w);
    const float *gain = head < a.heads ? a.turn.q_gain : a.turn.k_gain;
    if (head < a.turned) {
      if (gain) {
        auto mean = [&](float eps) {
          float sum = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; e++) sum = fmaf(u[e], u[e], fmaf(w[e], w[e], sum));
          return head_sum(there ? sum : 0.0f, per) / hd + eps;
        };
        float square = mean(a.turn.eps);
        if (!H && !(square >= 0x1p-100f && square < INFINITY)) {  // (squares past f32 on either side: of the values, scaled)
          const float scale = square < 1.0f ? 0x1p96f : 0x1p-96f;
          u *= scale, w *= scale;
          square = mean(a.turn.eps * scale * scale);
        }
        const float r = 1.0f / sqrtf(square);
        u *= r * raw4(gain + first), w *= r * raw4(gain + second);
      }
      if (turns) {
        if (a.turn.pairs) {
          const floatx4 x = u, z = w;
          u = floatx4{x[0] * c[0] - x[1] * s[0], x[1] * c[0] + x[0] * s[0], x[2] * c[1] - x[3] * s[1], x[3] * c[1] + x[2] * s[1]};
          w = floatx4{z[0] * c[2] - z[1] * s[2], z[1] * c[2] + z[0] * s[2], z[2] * c[3] - z[3] * s[3], z[3] * c[3] + z[2] * s[3]};
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float x = u[e], z = w[e];
            u[e] = x * c[e] - z * s[e], w[e] = z * c[e] + x * s[e];
          }
        }
      }
    }
    if (there) store4(a.y, to + first, a.out16, u), store4(a.y, to + second, a.out16, w);
  }
}

__device__ __forceinline__ void norm_row(const NormArgs &a, size_t row, int position, int tid, int threads) {
  if (a.in16) norm_heads<true>(a, row, position, tid, threads);
  else norm_heads<false>(a, row, position, tid, threads);
}

__global__ __launch_bounds__(NORM_THREADS) void norm_kernel(NormArgs a) {
  const int row = blockIdx.x, b = row / a.rows, i = row - b * a.rows;
  if (a.count && i >= a.count[b]) return;
  const int n = min(max(a.n[b], 0), 1 << 24);
  const int depth = a.mask ? depth_of(a.mask + (size_t)b * a.mask_stride + (size_t)i * a.words, i) : i;
  norm_row(a, row, n + depth, threadIdx.x, NORM_THREADS);
}

struct AppendArgs {
  Turn turn;
  const void *k, *v;
  size_t stride;
  int in16;
  const int32_t *n, *count, *path;
  int batch, rows, tiles;  // tiles: that a sequence's rows can reach
  int32_t *n_out;
  Pages pages;
  unsigned tile_blocks;  // workgroups of tiles; those after them norm and rotate the queries' rows
  NormArgs q;
};

// The largest of 16 lanes' pairs of 16-bit numbers.
__device__ __forceinline__ u16x2 max16(u16x2 v) {
  auto take = [](u16x2 a, int b) { return __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, b)); };
  v = take(v, xlane::dpp<xlane::XOR1>(__builtin_bit_cast(int, v)));
  v = take(v, xlane::dpp<xlane::XOR2>(__builtin_bit_cast(int, v)));
  v = take(v, xlane::dpp<xlane::HALF_MIRROR>(__builtin_bit_cast(int, v)));
  return take(v, xlane::dpp<xlane::MIRROR>(__builtin_bit_cast(int, v)));
}
// Two f16 values as numbers in the order of their magnitudes, the positive one of two first; no finite numbers last.
__device__ __forceinline__ u16x2 order2(uint32_t w) {
  return __builtin_bit_cast(u16x2, ((w << 1) & 0xfffefffeu) | ((~w >> 15) & 0x00010001u));
}
// Q4_0's factor of 32 values whose largest in that order is `top`: d = m / -8 rounded to f16 (exactly, where it is no
// subnormal; a zero is +0); NaN where one of them is no finite number.
__device__ __forceinline__ _Float16 factor_of(uint32_t top) {
  if (top >= 0xf800u) return __builtin_bit_cast(_Float16, (uint16_t)0x7e00);
  const float m = (float)__builtin_bit_cast(_Float16, (uint16_t)(top >> 1));
  return (_Float16)(m * (top & 1 ? -0.125f : 0.125f)) + (_Float16)0;
}
// 1 / d, or zero, with which every value is nibble 8.
__device__ __forceinline__ float inverse_of(_Float16 d) {
  const float f = (float)d;
  return f != 0.0f ? __builtin_amdgcn_rcpf(f) : 0.0f;
}
// floor(x / d + 8.5) within 0 .. 15.  x and d are f16, so a quotient that is not at a border k + 1/2 is at least 2^-12 from
// it, and one at the border has to go up: a nudge of 2^-14, beside the reciprocal's error of 2^-20, gives every value the
// nibble of the exact quotient.
__device__ __forceinline__ uint32_t nibble(float x, float inverse) {
  return (uint32_t)__builtin_amdgcn_fmed3f(fmaf(x, inverse, 8.5f + 0x1p-14f), 0.0f, 15.0f);
}

// 8 values of a row as they stand.
template <typename T>
struct Eight {
  typename Four<T>::type a, b;
};
template <typename T>
__device__ __forceinline__ Eight<T> raw8(const T *p) { return Eight<T>{raw4(p), raw4(p + 4)}; }
__device__ __forceinline__ float at8(const Eight<float> &x, int e) { return e < 4 ? x.a[e] : x.b[e - 4]; }
__device__ __forceinline__ float at8(const Eight<_Float16> &x, int e) {
  return (float)__builtin_bit_cast(half4, e < 4 ? x.a : x.b)[e & 3];
}
__device__ __forceinline__ uint32_t pair_at(const float *p) {
  typedef floatx2 any __attribute__((aligned(4)));
  const floatx2 f = *(const any *)p;
  return pack2(f[0], f[1]);
}
__device__ __forceinline__ uint32_t pair_at(const _Float16 *p) { return *(const uint32_t *)p; }

// x in f32.  (The compiler would turn a conversion to f16 by way of f32 into one in some 20 integer instructions.)
__device__ __forceinline__ float single(double x) {
  float f = (float)x;
  asm("" : "+v"(f));
  return f;
}

// Where the rows of a tile's new positions are: of position j of the tile, in the sequence's rows, or -1.
struct Rows {
  const int32_t *path;
  int first, end, rows;  // of the tile's first position, in the sequence; one past the last that is stored, from the tile's first
  __device__ __forceinline__ int operator()(int j) const {
    const int r = first + j;
    if (r < 0 || j >= end) return -1;
    if (!path) return r;
    const int p = path[r];
    return (uint32_t)p < (uint32_t)rows ? p : -1;
  }
};

// How a key is turned: not at all, by values of any lane (read again) or by values of the same one (the head's halves, of 64
// and 128 values).
enum { PLAIN, ANY, HALVES };

// New keys of 16 positions of a tile, by one wavefront, whose lanes hold them as the tile's words do (pages.h): a position's in
// the four lanes of its row.  They are normed and rotated in 64 bits: the last bits of f32 would cross a border of f16 for
// one of 1e3 values and of 4 bits for one of 1e5; as it is, a row leaves the words of its exact values.
template <typename T, int Z, bool Q4, int TURN>
__device__ __forceinline__ void append_k(const AppendArgs &a, const Rows &rows, const T *k0, uint32_t *out, int j0, int u) {
  constexpr int hd = 32 * Z;
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15, row = rows(16 * u + m);
  const T *k = k0 + (size_t)max(row, 0) * a.stride;
  const float *table = a.turn.table ? a.turn.table + (size_t)min(max(j0 + 16 * u + m, 0), a.turn.positions - 1) * a.turn.rot : nullptr;
  Eight<T> raw[Z];
#pragma unroll
  for (int c = 0; c < Z; c++) raw[c] = raw8(k + 32 * c + 8 * g);
  uint32_t w[Z][4];  // pairs of halfs
  if constexpr (TURN == PLAIN) {
#pragma unroll
    for (int c = 0; c < Z; c++) {
      const u32x2 p = pairs4(raw[c].a), q = pairs4(raw[c].b);
      w[c][0] = p[0], w[c][1] = p[1], w[c][2] = q[0], w[c][3] = q[1];
    }
  } else {
    double r = 1.0;
    if (a.turn.k_gain) {
      double sum = 0.0, more = 0.0;
#pragma unroll
      for (int c = 0; c < Z; c++)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const double x = at8(raw[c], e), y = at8(raw[c], e + 1);
          sum = fma(x, x, sum), more = fma(y, y, more);
        }
      sum = xlane::bit4(sum + more, xlane::Add{});
      sum = xlane::bit5(sum, xlane::Add{});
      r = 1.0 / sqrt(sum / hd + (double)a.turn.eps);
    }
    auto normed = [&](float y, float gain) { return a.turn.k_gain ? (double)y * r * (double)gain : (double)y; };
    auto gain4 = [&](int d) { return a.turn.k_gain ? raw4(a.turn.k_gain + d) : floatx4{}; };
    if constexpr (TURN == HALVES) {
#pragma unroll
      for (int c = 0; c < Z / 2; c++)
#pragma unroll
        for (int y = 0; y < 2; y++) {
          const int d = 32 * c + 8 * g + 4 * y;
          const floatx4 cs = raw4(table + d), sn = raw4(table + hd / 2 + d), ga = gain4(d), gb = gain4(hd / 2 + d);
          float p[4], q[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const double x = normed(at8(raw[c], 4 * y + e), ga[e]), z = normed(at8(raw[c + Z / 2], 4 * y + e), gb[e]);
            p[e] = single(x * cs[e] - z * sn[e]), q[e] = single(z * cs[e] + x * sn[e]);
          }
          w[c][2 * y] = pack2(p[0], p[1]), w[c][2 * y + 1] = pack2(p[2], p[3]);
          w[c + Z / 2][2 * y] = pack2(q[0], q[1]), w[c + Z / 2][2 * y + 1] = pack2(q[2], q[3]);
        }
    } else {
      const int half = a.turn.rot / 2;
#pragma unroll
      for (int c = 0; c < Z; c++)
#pragma unroll
        for (int y = 0; y < 2; y++) {
          const int d = 32 * c + 8 * g + 4 * y;
          const floatx4 gain = gain4(d);
          double x[4];
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = normed(at8(raw[c], 4 * y + e), gain[e]);
          if (d < a.turn.rot) {
            if (a.turn.pairs) {
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const double cs = table[(d + e) / 2], sn = table[half + (d + e) / 2], p = x[e], q = x[e + 1];
                x[e] = p * cs - q * sn, x[e + 1] = q * cs + p * sn;
              }
            } else {
              const bool low = d < half;
              const int other = low ? d + half : d - half, i = low ? d : d - half;
              const floatx4 f = load4(k, other, sizeof(T) == 2), cs = raw4(table + i), sn = raw4(table + half + i), go = gain4(other);
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const double q = normed(f[e], go[e]);
                x[e] = low ? x[e] * cs[e] - q * sn[e] : x[e] * cs[e] + q * sn[e];
              }
            }
          }
          w[c][2 * y] = pack2(single(x[0]), single(x[1])), w[c][2 * y + 1] = pack2(single(x[2]), single(x[3]));
        }
    }
  }

  if constexpr (!Q4) {
    if (row >= 0)
#pragma unroll
      for (int c = 0; c < Z; c++)
        *(u32x4 *)((_Float16 *)out + ((2 * c + u) * 64 + lane) * 8) = u32x4{w[c][0], w[c][1], w[c][2], w[c][3]};
  } else {
    uint16_t *const kd = (uint16_t *)(out + 4 * hd);
#pragma unroll
    for (int c = 0; c < Z; c++) {
      u16x2 top = order2(w[c][0]);
#pragma unroll
      for (int e = 1; e < 4; e++) top = __builtin_elementwise_max(top, order2(w[c][e]));
      uint32_t t = max((uint32_t)top[0], (uint32_t)top[1]);
      t = xlane::bit4(t, [](uint32_t x, uint32_t y) { return max(x, y); });
      t = xlane::bit5(t, [](uint32_t x, uint32_t y) { return max(x, y); });
      const _Float16 d = factor_of(t);
      const float inv = inverse_of(d);
      uint32_t word = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) word |= nibble((float)__builtin_bit_cast(half2, w[c][e / 2])[e & 1], inv) << nibble_of(e);
      if (row >= 0) {
        out[word_at(2 * c + u, lane, 2 * Z)] = word;
        // (position 16u + m is element 4u + m % 4 of group m / 4)
        if (g == 0) kd[((m >> 2) * Z + c) * 8 + 4 * u + (m & 3)] = __builtin_bit_cast(uint16_t, d);
      }
    }
  }
}

// New values of a tile, by one wavefront, whose lanes hold pairs of neighbouring values of 8 positions each.
template <typename T, int Z, bool Q4>
__device__ __forceinline__ void append_v(const AppendArgs &a, const Rows &rows, const T *v0, uint32_t *out) {
  constexpr int hd = 32 * Z;
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  int row[8];
  uint32_t v[8][Z], there = 0;  // of this lane's positions, those that are stored
#pragma unroll
  for (int e = 0; e < 8; e++) {
    row[e] = rows(position_of(g, e));
    there |= row[e] >= 0 ? 1u << e : 0u;
  }
#pragma unroll
  for (int e = 0; e < 8; e++)
#pragma unroll
    for (int c = 0; c < Z; c++) v[e][c] = pair_at(v0 + (size_t)max(row[e], 0) * a.stride + 32 * c + 2 * m);
  if constexpr (!Q4) {
    _Float16 *const values = (_Float16 *)out + 32 * hd;
#pragma unroll
    for (int c = 0; c < Z; c++)
#pragma unroll
      for (int x = 0; x < 2; x++) {
        _Float16 *const p = values + ((2 * c + x) * 64 + lane) * 8;
        if (there == 0xff) {
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = __builtin_amdgcn_perm(v[2 * e + 1][c], v[2 * e][c], x ? 0x07060302u : 0x05040100u);
          *(u32x4 *)p = w;
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (there >> e & 1) ((uint16_t *)p)[e] = (uint16_t)(v[e][c] >> 16 * x);
        }
      }
  } else {
    uint16_t *const vd = (uint16_t *)(out + 8 * hd + hd / 2);
    uint32_t *const words = out + 4 * hd + hd / 2;
    uint32_t keep = 0, old[2 * Z];  // nibbles of a word that stay, and the words before
#pragma unroll
    for (int e = 0; e < 8; e++) keep |= there >> e & 1 ? 0u : 15u << nibble_of(e);
#pragma unroll
    for (int x = 0; x < 2 * Z; x++) old[x] = 0;
    if (there && keep)
#pragma unroll
      for (int x = 0; x < 2 * Z; x++) old[x] = words[word_at(x, lane, 2 * Z)];
#pragma unroll
    for (int c = 0; c < Z; c++) {
      uint32_t w[2] = {0, 0};
      _Float16 d[8];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        // (the pair of positions e and e + 1, side by side)
        const u16x2 o = order2(v[e][c]), p = order2(v[e + 1][c]);
        const u16x2 top = max16(u16x2{(uint16_t)max(o[0], o[1]), (uint16_t)max(p[0], p[1])});
#pragma unroll
        for (int y = 0; y < 2; y++) {
          d[e + y] = factor_of(top[y]);
          const float inv = inverse_of(d[e + y]);
          const half2 x = __builtin_bit_cast(half2, v[e + y][c]);
          w[0] |= nibble((float)x[0], inv) << nibble_of(e + y), w[1] |= nibble((float)x[1], inv) << nibble_of(e + y);
        }
      }
      _Float16 *const f = (_Float16 *)vd + (g * Z + c) * 8;
      if (there == 0xff) {
        if (m == c) *(half8 *)f = half8{d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7]};
      } else if (m < 8 && there >> m & 1) {  // (lane m the one of element m)
        _Float16 mine = d[0];
#pragma unroll
        for (int e = 1; e < 8; e++) mine = m == e ? d[e] : mine;
        f[m] = mine;
      }
      if (there)
#pragma unroll
        for (int x = 0; x < 2; x++) words[word_at(2 * c + x, lane, 2 * Z)] = (old[2 * c + x] & keep) | (w[x] & ~keep);
    }
  }
}

// Tiles, and behind them the queries' rows.  A tile's words are put together in registers and written whole wherever all of
// their positions are new; keys of 16 positions and values of 32 go to wavefronts of their own, since one wavefront for a whole
// tile had its reads wait for each other three times over (16 tokens of 8 heads of 128 into 4 bits: 30 us, 8.4 now; 8192 rows:
// 132, 51 now).  Those 8192 rows, f16 with 32 query heads on the way, move 170 MB, 3.3 TB/s; without the queries they take 21 us (18
// into f16 pages) for 43 MB: vector instructions, 12 a value of K and 18 of V for factors and nibbles, and 11 of K, at half the
// rate, for the norm and rotation in 64 bits.
template <typename T, int Z, bool Q4, int TURN>
__global__ __launch_bounds__(256, 4) void append_kernel(AppendArgs a) {
  if (blockIdx.x >= a.tile_blocks) {
    const int row = blockIdx.x - a.tile_blocks, b = row / a.rows, i = row - b * a.rows;
    if (a.count && i >= a.count[b]) return;
    const int n = min(max(a.n[b], 0), a.pages.room);
    norm_row(a.q, row, n + i, threadIdx.x, 256);
    return;
  }
  // A wavefront per (sequence, tile, its values or half of its keys, key head), heads first.
  const unsigned heads = a.pages.kv_heads, per = a.tiles * 3 * heads;
  const unsigned wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = wave / per, rest = wave - b * per, t = rest / (3 * heads), part = rest / heads - 3 * t, kh = rest % heads;
  if (b >= a.batch) return;
  const int n = min(max(a.n[b], 0), a.pages.room), count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows;
  const int end = min(n + count, a.pages.room);
  if (a.n_out && rest == 0 && (threadIdx.x & 63) == 0) a.n_out[b] = end;
  const int tile = n / TILE + t, j0 = TILE * tile, u = part - 1;
  if (part ? j0 + 16 * u >= end || j0 + 16 * u + 16 <= n : j0 >= end) return;
  uint32_t *out = tile_at(a.pages, Q4, b, tile, kh);
  if (!out) return;
  const Rows rows{a.path ? a.path + (size_t)b * a.rows : nullptr, j0 - n, end - j0, a.rows};
  const size_t from = (size_t)b * a.rows * a.stride + (size_t)kh * 32 * Z;
  if (part) append_k<T, Z, Q4, TURN>(a, rows, (const T *)a.k + from, out, j0, u);
  else append_v<T, Z, Q4>(a, rows, (const T *)a.v + from, out);
}

// One step of turning four lanes' four words: words i and i + D, of which lane and partner (D apart) exchange one each.
template <int D>
__device__ __forceinline__ void swap_pairs(uint32_t (&w)[4], int m) {
  const bool high = m & D;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (i & D) continue;
    const uint32_t got = xlane::dpp<D == 1 ? xlane::XOR1 : xlane::XOR2>((int)(high ? w[i] : w[i + D]));
    if (high) w[i] = got;
    else w[i + D] = got;
  }
}

struct ReadArgs {
  Pages pages;
  const int32_t *n, *count;
  int batch, rows, tiles, out16;
  void *k, *v;
  size_t stride;
};

// Keys and values out of a tile, in the order of its words: a wavefront reads a tile of a head whole and stores 16 bytes of a
// row a lane (f16; values are turned for it).  8192 rows of 8 heads of 128 out of 4 bits into f16: 15 us, 2.9 TB/s (16.4 with values
// stored pair by pair); the launch, a tile's chain of length, page and words, and one wave of workgroups.
template <int Z, bool Q4>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  const unsigned wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), per = (unsigned)a.tiles * a.pages.kv_heads;
  const int b = wave / per, rest = wave % per, t = rest / a.pages.kv_heads, kh = rest % a.pages.kv_heads;
  if (b >= a.batch) return;
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  constexpr int hd = 32 * Z;
  const int n = min(max(a.n[b], 0), a.pages.room), count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows, end = n + count;
  // (rows past the last position of a sequence are zeros, as those of pages that are not there)
  const int j0 = n / TILE * TILE + TILE * t;
  if (j0 >= end) return;
  const uint32_t *in = j0 < a.pages.room ? tile_at(a.pages, Q4, b, j0 / TILE, kh) : nullptr;
  const size_t row0 = (size_t)b * a.rows;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int j = j0 + 16 * u + m;
    if (j < n || j >= end) continue;
    const size_t to = (row0 + (j - n)) * a.stride + (size_t)kh * hd + 8 * g;
#pragma unroll
    for (int c = 0; c < Z; c++) {
      floatx4 f[2] = {};
      if (in) {
        if constexpr (Q4) {
          const uint32_t w = in[word_at(2 * c + u, lane, 2 * Z)];
          const float d = (float)__builtin_bit_cast(_Float16, ((const uint16_t *)(in + 4 * hd))[((m >> 2) * Z + c) * 8 + 4 * u + (m & 3)]);
#pragma unroll
          for (int e = 0; e < 8; e++) f[e / 4][e % 4] = (float)((int)(w >> nibble_of(e) & 15) - 8) * d;
        } else {
          const half8 h = *(const half8 *)((const _Float16 *)in + ((2 * c + u) * 64 + lane) * 8);
#pragma unroll
          for (int e = 0; e < 8; e++) f[e / 4][e % 4] = (float)h[e];
        }
      }
      if (a.out16) {
        typedef u32x4 any __attribute__((aligned(4)));
        *(any *)((_Float16 *)a.k + to + 32 * c) = u32x4{pack2(f[0][0], f[0][1]), pack2(f[0][2], f[0][3]), pack2(f[1][0], f[1][1]), pack2(f[1][2], f[1][3])};
      } else {
        store4(a.k, to + 32 * c, 0, f[0]), store4(a.k, to + 32 * c + 4, 0, f[1]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < Z; c++) {
    float f[2][8] = {};
    if (in) {
#pragma unroll
      for (int x = 0; x < 2; x++) {
        if constexpr (Q4) {
          const uint32_t w = in[4 * hd + hd / 2 + word_at(2 * c + x, lane, 2 * Z)];
          const half8 d = *(const half8 *)((const _Float16 *)(in + 8 * hd + hd / 2) + (g * Z + c) * 8);
#pragma unroll
          for (int e = 0; e < 8; e++) f[x][e] = (float)((int)(w >> nibble_of(e) & 15) - 8) * (float)d[e];
        } else {
          const half8 h = *(const half8 *)((const _Float16 *)in + 32 * hd + ((2 * c + x) * 64 + lane) * 8);
#pragma unroll
          for (int e = 0; e < 8; e++) f[x][e] = (float)h[e];
        }
      }
    }
    if (a.out16) {
      // Four lanes' pairs of four positions turned, so that lane m has 8 values of position 16i + 4g + m % 4.
#pragma unroll
      for (int i = 0; i < 2; i++) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = pack2(f[0][4 * i + e], f[1][4 * i + e]);
        swap_pairs<1>(w, m), swap_pairs<2>(w, m);
        const int j = j0 + position_of(g, 4 * i + m % 4);
        typedef u32x4 any __attribute__((aligned(4)));
        if (j >= n && j < end) *(any *)((_Float16 *)a.v + (row0 + (j - n)) * a.stride + (size_t)kh * hd + 32 * c + m / 4 * 8) = u32x4{w[0], w[1], w[2], w[3]};
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int j = j0 + position_of(g, e);
        typedef floatx2 any __attribute__((aligned(4)));
        if (j >= n && j < end) *(any *)((float *)a.v + (row0 + (j - n)) * a.stride + (size_t)kh * hd + 32 * c + 2 * m) = floatx2{f[0][e], f[1][e]};
      }
    }
  }
}

template <typename T, int Z, bool Q4>
void append_launch(wh_ctx *ctx, const AppendArgs &a, unsigned blocks) {
  if (!a.turn.k_gain && !a.turn.table) return wh_launch(ctx, (append_kernel<T, Z, Q4, PLAIN>), blocks, 256, 0, a);
  if constexpr (Z % 2 == 0)
    if (a.turn.table && a.turn.rot == 32 * Z && !a.turn.pairs) return wh_launch(ctx, (append_kernel<T, Z, Q4, HALVES>), blocks, 256, 0, a);
  wh_launch(ctx, (append_kernel<T, Z, Q4, ANY>), blocks, 256, 0, a);
}
template <typename T, bool Q4>
void append_z(wh_ctx *ctx, const AppendArgs &a, unsigned blocks) {
  switch (a.pages.hd / 32) {
    case 1: return append_launch<T, 1, Q4>(ctx, a, blocks);
    case 2: return append_launch<T, 2, Q4>(ctx, a, blocks);
    case 3: return append_launch<T, 3, Q4>(ctx, a, blocks);
    default: return append_launch<T, 4, Q4>(ctx, a, blocks);
  }
}
template <bool Q4>
void read_z(wh_ctx *ctx, const ReadArgs &a, unsigned blocks) {
  switch (a.pages.hd / 32) {
    case 1: return wh_launch(ctx, (read_kernel<1, Q4>), blocks, 256, 0, a);
    case 2: return wh_launch(ctx, (read_kernel<2, Q4>), blocks, 256, 0, a);
    case 3: return wh_launch(ctx, (read_kernel<3, Q4>), blocks, 256, 0, a);
    default: return wh_launch(ctx, (read_kernel<4, Q4>), blocks, 256, 0, a);
  }
}

int heads_check(wh_ctx *ctx, const char *what, const wh_heads *h) {
  if (!h || h->heads <= 0 || h->heads > ATTEND_HEADS || h->kv_heads <= 0 || h->heads % h->kv_heads || h->hd <= 0 || h->hd > 256 || h->hd % 8)
    return wh_fail(ctx, WH_EARG, "%s: bad heads (%d, %d of keys, of %d values)", what, h ? h->heads : 0, h ? h->kv_heads : 0, h ? h->hd : 0);
  if ((h->q_gain || h->k_gain) && !(h->eps >= 0.0f && h->eps < INFINITY)) return wh_fail(ctx, WH_EARG, "%s: norms with eps %g", what, h->eps);
  if (h->table && (h->positions <= 0 || h->positions > 1 << 24 || h->rot <= 0 || h->rot > h->hd || h->rot % 8))
    return wh_fail(ctx, WH_EARG, "%s: a rotation of %d values of %d by %d positions", what, h->rot, h->hd, h->positions);
  if (((uintptr_t)h->q_gain | (uintptr_t)h->k_gain | (uintptr_t)h->table) % 4)
    return wh_fail(ctx, WH_EARG, "%s: gains and the table must be 4-byte aligned", what);
  return WH_OK;
}
Turn turn_of(const wh_heads *h) { return Turn{h->q_gain, h->k_gain, h->eps, h->table, h->table ? h->positions : 0, h->table ? h->rot : 0, h->pairs}; }
int lanes_of(int hd) {
  int per = 1;
  while (8 * per < hd) per *= 2;
  return per;
}

}  // namespace

size_t page_bytes(int type, int page, int kv_heads, int hd) {
  if ((type != WH_F16 && type != WH_Q4_0) || page < 32 || page > 256 || (page & (page - 1)) || kv_heads <= 0 || kv_heads > ATTEND_HEADS ||
      hd <= 0 || hd > 128 || hd % 32)
    return 0;
  return (size_t)4 * tile_words(type == WH_Q4_0, hd) * (page / TILE) * kv_heads;
}

int pages_check(wh_ctx *ctx, const char *what, const wh_pages *p) {
  if (!p || !page_bytes(p->type, p->page, p->kv_heads, p->hd))
    return wh_fail(ctx, WH_EARG, "%s: pages of %d positions of %d heads of %d values of type %d are not supported", what, p ? p->page : 0,
                   p ? p->kv_heads : 0, p ? p->hd : 0, p ? p->type : 0);
  if (!p->pool || !p->table || p->pages <= 0 || p->table_cols <= 0 || (int64_t)p->table_cols * p->page > 1 << 24)
    return wh_fail(ctx, WH_EARG, "%s: a pool of pages and tables of up to 2^24 positions are needed (%d pages, %d columns)", what, p->pages,
                   p->table_cols);
  if (p->table_stride && p->table_stride < (size_t)p->table_cols)
    return wh_fail(ctx, WH_EARG, "%s: tables of %d pages %zu apart", what, p->table_cols, p->table_stride);
  if ((uintptr_t)p->pool % 16 || (uintptr_t)p->table % 4)
    return wh_fail(ctx, WH_EARG, "%s: the pool must be 16-byte aligned, the tables 4-byte", what);
  return WH_OK;
}

pages::Pages pages_of(const wh_pages *p) {
  int shift = 5;
  while (1 << shift < p->page) shift++;
  return Pages{(uint32_t *)p->pool, p->table, p->table_stride, p->pages, shift, p->table_cols * p->page, p->kv_heads, p->hd,
               page_bytes(p->type, p->page, p->kv_heads, p->hd) / 4};
}

int launch_head_norm(wh_ctx *ctx, const wh_tree *t, const wh_heads *h, const void *x, size_t stride, int in16, void *y, size_t y_stride,
                     int out16) {
  if (int rc = tree_check(ctx, "head norm", t)) return rc;
  if (int rc = heads_check(ctx, "head norm", h)) return rc;
  if (!x || !y) return wh_fail(ctx, WH_EARG, "head norm: rows and their output are needed");
  const size_t least = (size_t)(h->heads + 2 * h->kv_heads) * h->hd;
  if (stride < least || stride > (size_t)1 << 31 || y_stride < least || y_stride > (size_t)1 << 31)
    return wh_fail(ctx, WH_EARG, "head norm: rows of %zu values %zu and %zu apart", least, stride, y_stride);
  if (((uintptr_t)x | (uintptr_t)y) % 4 || (in16 && stride % 2) || (out16 && y_stride % 2))
    return wh_fail(ctx, WH_EARG, "head norm: buffers and rows must be 4-byte aligned");
  const bool same = x == y;
  if (same && (!in16 != !out16 || stride != y_stride)) return wh_fail(ctx, WH_EARG, "head norm: rows in their own place keep type and stride");
  const size_t nodes = (size_t)t->batch * t->rows, in = in16 ? 2 : 4, out = out16 ? 2 : 4;
  if (!same && rows_meet(x, least * in, stride * in, y, least * out, y_stride * out, nodes))
    return wh_fail(ctx, WH_EARG, "head norm: the output overlaps the rows");
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "head norm: %s", hipGetErrorString(e));
  const NormArgs a{turn_of(h), x, stride, y, y_stride, t->n, t->count, t->mask, t->mask_stride, t->rows, (t->rows + 31) / 32, h->heads,
                   h->heads + h->kv_heads, h->heads + (same ? 1 : 2) * h->kv_heads, h->hd, lanes_of(h->hd), in16 != 0, out16 != 0};
  ProfScope prof(ctx, "head_norm", 10.0 * nodes * a.turned * h->hd, (double)nodes * a.all * h->hd * (in + out));
  wh_launch(ctx, norm_kernel, (unsigned)nodes, NORM_THREADS, 0, a);
  return wh_launched(ctx, "head norm");
}

int launch_page_append(wh_ctx *ctx, const wh_tree *t, const wh_heads *h, const void *q, const void *k, const void *v, size_t stride, int in16,
                       const int32_t *path, const int32_t *kept, const wh_pages *p, void *qo, size_t qo_stride, int out16, int32_t *n_out) {
  if (int rc = tree_check(ctx, "page append", t)) return rc;
  if (int rc = heads_check(ctx, "page append", h)) return rc;
  if (int rc = pages_check(ctx, "page append", p)) return rc;
  if (p->kv_heads != h->kv_heads || p->hd != h->hd)
    return wh_fail(ctx, WH_EARG, "page append: %d heads of %d values into pages of %d of %d", h->kv_heads, h->hd, p->kv_heads, p->hd);
  if (!k || !v || !q != !qo || (q && path)) return wh_fail(ctx, WH_EARG, "page append: k and v are needed, q with its output and without a path");
  const size_t least = (size_t)h->kv_heads * h->hd, qleast = (size_t)h->heads * h->hd;
  if (stride < (q ? qleast : least) || stride > (size_t)1 << 31 || (q && (qo_stride < qleast || qo_stride > (size_t)1 << 31)))
    return wh_fail(ctx, WH_EARG, "page append: rows of %zu values %zu apart, queries %zu", q ? qleast : least, stride, qo_stride);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)qo | (uintptr_t)path | (uintptr_t)kept | (uintptr_t)n_out) % 4 ||
      (in16 && stride % 2) || (q && out16 && qo_stride % 2))
    return wh_fail(ctx, WH_EARG, "page append: buffers and rows must be 4-byte aligned");
  if (q == qo && q && (!in16 != !out16 || stride != qo_stride))
    return wh_fail(ctx, WH_EARG, "page append: queries in their own place keep type and stride");
  const size_t nodes = (size_t)t->batch * t->rows;
  const int tiles = (t->rows + TILE - 2) / TILE + 1;
  const size_t waves = (size_t)t->batch * tiles * 3 * p->kv_heads, blocks = (waves + 3) / 4 + (q ? nodes : 0);
  if (blocks >= (size_t)1 << 24 || waves >= (size_t)1 << 31) return wh_fail(ctx, WH_EARG, "page append: %zu rows of %d heads in one call", nodes, p->kv_heads);
  const size_t in = in16 ? 2 : 4, out = out16 ? 2 : 4;
  auto over = [&](const void *x, size_t values) { return rows_meet(qo, qleast * out, qo_stride * out, x, values * in, stride * in, nodes); };
  if (q && ((q != qo && over(q, qleast)) || over(k, least) || over(v, least)))
    return wh_fail(ctx, WH_EARG, "page append: the queries' output overlaps the rows");
  auto counts = [&](const int32_t *x, size_t n) { return x && rows_meet(n_out, 4 * (size_t)t->batch, 4 * (size_t)t->batch, x, 4 * n, 4 * n, 1); };
  if (n_out && (counts(t->n, t->batch) || counts(t->count, t->batch) || counts(kept, t->batch) || counts(path, nodes)))
    return wh_fail(ctx, WH_EARG, "page append: n_out cannot be n, the numbers of rows or the paths");
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "page append: %s", hipGetErrorString(e));
  const int32_t *count = kept ? kept : t->count;
  const Turn turn = turn_of(h);
  const AppendArgs a{turn, k, v, stride, in16 != 0, t->n, count, path, t->batch, t->rows, tiles, n_out, pages_of(p), (unsigned)((waves + 3) / 4),
                     NormArgs{turn, q, stride, qo, qo_stride, t->n, count, nullptr, 0, t->rows, 0, h->heads, h->heads, h->heads, h->hd,
                              lanes_of(h->hd), in16 != 0, out16 != 0}};
  ProfScope prof(ctx, "page_append", 0.0, (double)nodes * (2 * least + (q ? qleast : 0)) * (in16 ? 2 : 4));
  if (p->type == WH_Q4_0) in16 ? append_z<_Float16, true>(ctx, a, blocks) : append_z<float, true>(ctx, a, blocks);
  else in16 ? append_z<_Float16, false>(ctx, a, blocks) : append_z<float, false>(ctx, a, blocks);
  return wh_launched(ctx, "page append");
}

int launch_page_read(wh_ctx *ctx, const wh_tree *t, const wh_pages *p, void *k, void *v, size_t stride, int out16) {
  if (int rc = tree_check(ctx, "page read", t)) return rc;
  if (int rc = pages_check(ctx, "page read", p)) return rc;
  if (!k || !v) return wh_fail(ctx, WH_EARG, "page read: rows for k and v are needed");
  if (stride < (size_t)p->kv_heads * p->hd || stride > (size_t)1 << 31)
    return wh_fail(ctx, WH_EARG, "page read: rows of %d values %zu apart", p->kv_heads * p->hd, stride);
  if (((uintptr_t)k | (uintptr_t)v) % 4 || (out16 && stride % 2)) return wh_fail(ctx, WH_EARG, "page read: buffers and rows must be 4-byte aligned");
  const int tiles = (t->rows + TILE - 2) / TILE + 1;
  const size_t waves = (size_t)t->batch * tiles * p->kv_heads, blocks = (waves + 3) / 4;
  if (blocks >= (size_t)1 << 24) return wh_fail(ctx, WH_EARG, "page read: %d rows of %d sequences in one call", t->rows, t->batch);
  const size_t out = out16 ? 2 : 4, values = (size_t)p->kv_heads * p->hd * out;
  if (rows_meet(k, values, stride * out, v, values, stride * out, (size_t)t->batch * t->rows))
    return wh_fail(ctx, WH_EARG, "page read: the rows of k and v overlap");
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "page read: %s", hipGetErrorString(e));
  const ReadArgs a{pages_of(p), t->n, t->count, t->batch, t->rows, tiles, out16 != 0, k, v, stride};
  ProfScope prof(ctx, "page_read", 0.0, (double)t->batch * t->rows * p->kv_heads * p->hd * 2 * (out16 ? 2 : 4));
  if (p->type == WH_Q4_0) read_z<true>(ctx, a, blocks);
  else read_z<false>(ctx, a, blocks);
  return wh_launched(ctx, "page read");
}
