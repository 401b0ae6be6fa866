// Sampling for a decoder step over trees of drafted tokens (include/wavo_hip.h): probabilities from logits, and the drafted
// tokens verified against them from given random numbers.
#include <algorithm>
#include <climits>

#include "internal.h"
#include "xlane.h"

namespace {

constexpr uint32_t NONE = 0xffffffffu;
constexpr int PT = 1024;  // threads of a row's workgroup

struct ProbsArgs {
  const void *logits;
  size_t ld;
  float *probs;
  size_t probs_ld;
  const float *temperature;
  const int32_t *count;
  int rows, vocab;
};

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
template <typename T>
struct Piece;
template <>
struct Piece<float> {
  typedef floatx4 any __attribute__((aligned(4)));
};
template <>
struct Piece<_Float16> {
  typedef half4 any __attribute__((aligned(2)));
};
// Values x .. x + 3 of a row of n; `past` for those that are not there.
template <typename T>
__device__ __forceinline__ floatx4 four_of(const T *p, int x, int n, float past) {
  if (x + 4 <= n) {
    const auto v = *(const typename Piece<T>::any *)(p + x);
    return floatx4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
  }
  floatx4 f;
#pragma unroll
  for (int e = 0; e < 4; e++) f[e] = x + e < n ? (float)p[x + e] : past;
  return f;
}

// The sum (maximum) over a workgroup's WV wavefronts of what each holds for itself.
template <int WV, class Op>
__device__ __forceinline__ float over_waves(float v, float *part, Op op, float none) {
  const int lane = threadIdx.x & 63;
  if (lane == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return xlane::butterfly(lane < WV ? part[lane] : none, op);
}

// A row per workgroup, its first HELD * 4096 values in registers from their one load to their store (longer rows' others are read
// three times, from the caches): the maximum, the exponents' sum, the quotients.  Sums in f32, of few terms a thread.
// HELD: as many pieces as 64 registers take without a spill, which is what two workgroups a compute unit leave a thread.  12 spill
// some and 13 more; with 11, 12 and 13 one row of 20000 f32 logits takes 5.5, 5.9 and 6.4 us, 384 rows 13, 14 and 16; of 51866
// (of which 11 read the last 6810 again) 7.8, 8.1 and 8.3, and 29, 30 and 35; of 131071 126, 126 and 129.  8 are better where they hold
// the whole row (12 us for 384 rows of 20000), and worse past that (133 of 131071).
// Many rows are bound by HBM: two workgroups a compute unit, one's loads beside the other's stores (384 rows of 51866: 159 MB in 29 us, some of them from the chip's cache).
// One row is bound by one compute unit's loads and stores of 200 KB each; in three passes over the row it took 21 us.
constexpr int HELD = 11;
template <typename T>
__global__ __launch_bounds__(PT, 8) void probs_kernel(ProbsArgs a) {
  __shared__ float tops[PT / 64], sums[PT / 64];
  __shared__ int first;
  constexpr int STEP = 4 * PT;
  const int row = blockIdx.x, b = row / a.rows, tid = threadIdx.x;
  const T *x = (const T *)a.logits + (size_t)row * a.ld;
  float *y = a.probs + (size_t)row * a.probs_ld;
  if (a.count && row - b * a.rows >= a.count[b]) return;
  const float t = a.temperature ? a.temperature[b] : 1.0f;
  if (tid == 0) first = INT_MAX;
  floatx4 v[HELD];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < HELD; i++) v[i] = i * STEP < a.vocab ? four_of(x, i * STEP + 4 * tid, a.vocab, -INFINITY) : floatx4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < HELD; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) top = fmaxf(top, v[i][e]);
  for (int at = HELD * STEP + 4 * tid; at < a.vocab; at += STEP) {
    const floatx4 f = four_of(x, at, a.vocab, -INFINITY);
#pragma unroll
    for (int e = 0; e < 4; e++) top = fmaxf(top, f[e]);
  }
  top = over_waves<PT / 64>(xlane::wave_max(top), tops, xlane::Max{}, -INFINITY);
  auto store = [&](int at, floatx4 f) {
    if (at + 4 <= a.vocab) {
      *(Piece<float>::any *)(y + at) = f;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (at + e < a.vocab) y[at + e] = f[e];
    }
  };
  if (!(t > 0.0f)) {  // all of it to the first maximum; NaN, if there is any or plus infinity (whose place is -1)
    int at = INT_MAX;
    for (int i = 4 * tid; i < a.vocab; i += STEP) {
      const floatx4 f = four_of(x, i, a.vocab, -INFINITY);
#pragma unroll
      for (int e = 0; e < 4; e++) at = min(at, !(f[e] < INFINITY) ? -1 : f[e] == top && top > -INFINITY ? i + e : INT_MAX);
    }
    if (at != INT_MAX) atomicMin(&first, at);
    __syncthreads();
    const int one = first;
    const float none = one < 0 ? NAN : 0.0f;
    for (int i = 4 * tid; i < a.vocab; i += STEP)
      store(i, floatx4{i == one ? 1.0f : none, i + 1 == one ? 1.0f : none, i + 2 == one ? 1.0f : none, i + 3 == one ? 1.0f : none});
    return;
  }
  // Half the difference, which is within f32 for any two values; and its factor, finite and no zero, so that what is left of minus
  // infinity is nothing at any temperature, and what is left of numbers at an infinite one all of them (2^-21 off, at f32's ends).
  const float base = top == -INFINITY ? 0.0f : -0.5f * top, k = fminf(fmaxf(2.88539008177792681f / t, 0x1p-149f), 3.402823466e38f);
  auto power = [&](floatx4 f) {
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] = __builtin_amdgcn_exp2f(fmaf(f[e], 0.5f, base) * k);
    return f;
  };
  float sum = 0.0f, more = 0.0f;
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    v[i] = power(v[i]);
    sum += v[i][0] + v[i][1], more += v[i][2] + v[i][3];
  }
  for (int at = HELD * STEP + 4 * tid; at < a.vocab; at += STEP) {
    const floatx4 f = power(four_of(x, at, a.vocab, -INFINITY));
    sum += f[0] + f[1], more += f[2] + f[3];
  }
  sum = over_waves<PT / 64>(xlane::wave_sum(sum + more), sums, xlane::Add{}, 0.0f);
  const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int i = 0; i < HELD; i++)
    if (i * STEP < a.vocab) store(i * STEP + 4 * tid, v[i] * scale);
  for (int at = HELD * STEP + 4 * tid; at < a.vocab; at += STEP) store(at, power(four_of(x, at, a.vocab, -INFINITY)) * scale);
}

struct SampleArgs {
  const float *p, *q, *u;
  const int32_t *count;
  const uint32_t *tokens, *mask;
  size_t mask_stride, ld;
  int rows, words, vocab;
  uint32_t *picks;
};

constexpr int ST = 1024;      // threads of a sequence's workgroup
constexpr int PIECES = 1024;  // runs of ids whose sums are kept

// What is left of N ids' probabilities x after rejections of their node's children's tokens, made anew from p and q whenever
// they are read.  With drafts y, w = max(0, w / Z - q) round by round (gone: 1 / Z); without, zero at the tokens (gone).
template <bool DRAFTS, int N, class Id>
__device__ __forceinline__ void left_of(const float (&x)[N], const float (&y)[N], double (&w)[N], const double *gone, int rounds, Id id) {
#pragma unroll
  for (int i = 0; i < N; i++) w[i] = x[i];
  for (int r = 0; r < rounds; r++) {
    const double z = gone[r];
    const int token = (int)z;
#pragma unroll
    for (int i = 0; i < N; i++) {
      if constexpr (DRAFTS) w[i] = fmax(w[i] * z - (double)y[i], 0.0);
      else w[i] = id(i) == token ? 0.0 : w[i];
    }
  }
}

// A sequence's walk by one workgroup.  What its tests need of p and q (a value per node, of its parent's rows) is gathered
// first, for all nodes side by side; a rejection that is followed by another child costs a pass over the rows for Z, and the
// draw one more, which leaves the sums of runs of ids behind, so that its place is looked for in one of them.  Everything in 64
// bits: random numbers are compared with sums of 1e5 values, whose last bits in f32 would move a place for one of 1e3.  The
// floor of the bytes (13 MB for 32 trees of 24 nodes over 51866 ids with drafts: 3 us) is far: a walk is a chain of passes,
// each of one compute unit's reads of two rows from the caches, 64-bit sums, and a meeting of 16 wavefronts.  Those trees take
// 31 to 41 us, by the tokens that were drawn, a chain of 8 nodes without drafts 14; with p and q looked up node by node and the
// draw's place by a second pass 104 and 29.
// Sums and products are rounded: of children that are all that is wanted none may be accepted, or Z be nothing before the last is
// looked at.  Then the draw falls on a child's token, and the walk goes on there (once for some 1e8 verifications), with the part of
// the random number that the draw did not use.
template <bool DRAFTS>
__global__ __launch_bounds__(ST) void sample_kernel(SampleArgs a) {
  __shared__ double part[ST / 64], sums[PIECES], gone[TREE_ROWS];
  __shared__ float mine[TREE_ROWS], drafted[TREE_ROWS], numbers[TREE_ROWS];
  __shared__ uint32_t tokens[TREE_ROWS], out[TREE_ROWS];
  __shared__ short parents[TREE_ROWS];
  __shared__ int found;
  __shared__ double left[2];
  constexpr int WV = ST / 64, BATCH = DRAFTS ? 5 : 7;  // BATCH: blocks of 256 ids that a wavefront loads at once
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows;
  if (count == 0) return;
  const size_t row0 = (size_t)b * a.rows;
  if (tid < count) {
    // A node's parent: the highest node below it that it sees.
    const int i = tid;
    int parent = i - 1;
    const float u = a.u[row0 + i];
    const uint32_t x = i ? a.tokens[row0 + i] : 0u;
    if (a.mask && i) {
      const uint32_t *m = a.mask + (size_t)b * a.mask_stride + (size_t)i * a.words;
      parent = -1;
      for (int w = (i - 1) / 32; w >= 0 && parent < 0; w--) {
        const uint32_t bits = m[w] & (w == i / 32 ? (1u << i % 32) - 1u : 0xffffffffu);
        if (bits) parent = 32 * w + 31 - __clz(bits);
      }
    }
    if (i && x >= (uint32_t)a.vocab) parent = -1;  // (no draft of this vocabulary)
    const size_t at = (row0 + max(parent, 0)) * a.ld + (x < (uint32_t)a.vocab ? x : 0u);
    mine[i] = a.p[at];
    if constexpr (DRAFTS) drafted[i] = a.q[at];
    numbers[i] = u, tokens[i] = x, parents[i] = (short)(i ? parent : -1), out[i] = NONE;
  }
  if (tid == 0) found = -1;
  __syncthreads();

  int at = 0, rounds = 0;  // the node, and how many of its children were rejected
  double total = 1.0, number = numbers[0];  // Z, and the draw's random number
  const float *p = a.p + row0 * a.ld, *q = DRAFTS ? a.q + row0 * a.ld : nullptr;
  auto enter = [&](int node) {
    at = node, rounds = 0, total = 1.0;
    p = a.p + (row0 + node) * a.ld, q = DRAFTS ? a.q + (row0 + node) * a.ld : nullptr;
  };
  // The rows of `at`, 256 ids (a wavefront's) at a time: f(piece, ids' weights).  A piece is `per` such blocks, one after the
  // other by one wavefront, and every wavefront takes every WV-th piece.
  const int blocks = (a.vocab + 255) / 256, per = (blocks + PIECES - 1) / PIECES, pieces = (blocks + per - 1) / per;
  auto pass = [&](auto f) {
    for (int n0 = 0; wave + WV * (n0 / per) < pieces; n0 += BATCH) {
      float x[4 * BATCH], y[4 * BATCH];
      double w[4 * BATCH];
      int piece[BATCH], block[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; i++) {
        piece[i] = wave + WV * ((n0 + i) / per), block[i] = piece[i] * per + (n0 + i) % per;
        if (piece[i] >= pieces) block[i] = blocks;  // (nothing there: zeros)
        const int id = 256 * block[i] + 4 * lane;
        *(floatx4 *)&x[4 * i] = four_of(p, id, a.vocab, 0.0f);
        if constexpr (DRAFTS) *(floatx4 *)&y[4 * i] = rounds ? four_of(q, id, a.vocab, 0.0f) : floatx4{};
      }
      left_of<DRAFTS>(x, y, w, gone, rounds, [&](int i) { return 256 * block[i / 4] + 4 * lane + i % 4; });
#pragma unroll
      for (int i = 0; i < BATCH; i++)
        if (block[i] < blocks) f(piece[i], (w[4 * i] + w[4 * i + 1]) + (w[4 * i + 2] + w[4 * i + 3]));
    }
  };
  // From `at` on, among the nodes from `from` on.
  int base = 0, from = 1;
  auto walk = [&] {
    while (base < count) {
      // The next child of `at`, among 64 nodes at a time.
      const int i0 = base + lane;
      const uint64_t any = __ballot(i0 >= from && i0 < count && parents[min(i0, count - 1)] == at);
      if (!any) {
        base += 64;
        continue;
      }
      const int i = base + (int)__builtin_ctzll(any);
      const int x = (int)tokens[i];
      if (DRAFTS && rounds && total < 0.0) {  // (Z of the rejections so far, wanted only now)
        double s = 0.0;
        pass([&](int, double w) { s += w; });
        s = xlane::wave_sum(s);
        if (lane == 0) part[wave] = s;
        __syncthreads();
        total = 0.0;
#pragma unroll
        for (int w = 0; w < WV; w++) total += part[w];
        __syncthreads();
      }
      if (!(total > 0.0)) break;  // nothing is left to accept
      from = i + 1;
      const float own[1] = {mine[i]}, draft[1] = {DRAFTS ? drafted[i] : 0.0f};
      double kept[1];
      left_of<DRAFTS>(own, draft, kept, gone, rounds, [&](int) { return x; });
      const double w = kept[0];
      if ((double)numbers[i] * (DRAFTS ? (double)drafted[i] : 1.0) * total < w) {
        if (tid == 0) out[at] = (uint32_t)x;
        enter(i);
        base = i / 64 * 64;
        continue;
      }
      __syncthreads();
      if (tid == 0) gone[rounds] = DRAFTS ? 1.0 / total : (double)x;
      __syncthreads();
      rounds++;
      total = DRAFTS ? -1.0 : total - w;
    }
  };
  // The id drawn at `at`, or -1.  How far the place is into the id's weight, and that, stay behind as `left`.
  auto draw = [&] {
    for (int attempt = 0; attempt < 2; attempt++) {
      __syncthreads();
      for (int i = tid; i < PIECES; i += ST) sums[i] = 0.0;
      __syncthreads();
      pass([&](int piece, double w) {
        w = xlane::wave_sum(w);
        if (lane == 0) sums[piece] += w;
      });
      __syncthreads();
      // Running sums of 16 pieces a lane, by every wavefront for itself.
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < PIECES / 64; i++) s += sums[PIECES / 64 * lane + i];
      double c = s;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const double o = __shfl_up(c, d);
        if (lane >= d) c += o;
      }
      const double all = __shfl(c, 63);
      if (!(all > 0.0)) {  // nothing left: from the node's probabilities themselves
        rounds = 0;
        continue;
      }
      const double place = number * all;
      if (wave == 0) {
        // The first lane, then its first piece, then the first id whose running sum is past the place; where last bits leave none,
        // the last one of any weight.
        const uint64_t over = __ballot(s > 0.0 && c > place), some = __ballot(s > 0.0);
        const int l = over ? (int)__builtin_ctzll(over) : 63 - (int)__clzll(some);
        double before = __shfl(c - s, l);
        int piece = -1, last = 0;
        for (int i = 0; i < PIECES / 64 && piece < 0; i++) {
          const int k = PIECES / 64 * l + i;
          if (k >= pieces) break;
          if (sums[k] > 0.0) last = k;
          if (sums[k] > 0.0 && before + sums[k] > place) piece = k;
          else before += sums[k];
        }
        if (piece < 0) piece = last, before -= sums[last];
        int hit = -1, tail = -1;
        double past = 1.0, weight = 1.0;
        for (int k = piece * per; k < min((piece + 1) * per, blocks) && hit < 0; k++) {
          const int id = 256 * k + 4 * lane;
          float x[4], y[4];
          *(floatx4 *)x = four_of(p, id, a.vocab, 0.0f);
          *(floatx4 *)y = DRAFTS && rounds ? four_of(q, id, a.vocab, 0.0f) : floatx4{};
          double w[4];
          left_of<DRAFTS>(x, y, w, gone, rounds, [&](int e) { return id + e; });
          const double r = (w[0] + w[1]) + (w[2] + w[3]);
          double run = r;
#pragma unroll
          for (int d = 1; d < 64; d *= 2) {
            const double o = __shfl_up(run, d);
            if (lane >= d) run += o;
          }
          double here = before + (run - r), below = 0.0, share = 1.0;
          int own = -1, end = -1;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if (w[e] > 0.0) end = id + e;
            if (own < 0 && w[e] > 0.0 && here + w[e] > place) own = id + e, below = here, share = w[e];
            here += w[e];
          }
          const uint64_t hits = __ballot(own >= 0), ends = __ballot(end >= 0);
          if (hits) {
            const int x = (int)__builtin_ctzll(hits);
            hit = __shfl(own, x), past = place - __shfl(below, x), weight = __shfl(share, x);
          }
          if (ends) tail = __shfl(end, 63 - (int)__clzll(ends));
          before += __shfl(run, 63);
        }
        if (lane == 0) found = hit >= 0 ? hit : tail, left[0] = past, left[1] = weight;
      }
      __syncthreads();
      return found;
    }
    return -1;
  };
  // A draw that falls on the token of a child, though none was accepted, goes on there: wh_tree_accept will.
  for (;;) {
    walk();
    const int id = draw();
    if (tid == 0) out[at] = (uint32_t)id;
    int next = -1;
    for (int i0 = at / 64 * 64; id >= 0 && i0 < count && next < 0; i0 += 64) {
      const int i = min(i0 + lane, count - 1);
      const uint64_t any = __ballot(i > at && parents[i] == at && tokens[i] == (uint32_t)id);
      if (any) next = i0 + (int)__builtin_ctzll(any);
    }
    if (next < 0) break;
    number = fmin(fmax(left[0] / left[1], 0.0), 0x1.fffffffffffffp-1);
    enter(next);
    base = next / 64 * 64, from = next + 1;
  }
  __syncthreads();
  if (tid < count) a.picks[row0 + tid] = out[tid];
}

}  // namespace

int launch_logit_probs(wh_ctx *ctx, const wh_tree *t, const void *logits, size_t ld, int f16, int vocab, const float *temperature, float *probs,
                       size_t probs_ld) {
  if (int rc = tree_check(ctx, "logit probabilities", t)) return rc;
  if (!logits || !probs || vocab <= 0 || vocab > 1 << 28 || ld < (size_t)vocab || probs_ld < (size_t)vocab)
    return wh_fail(ctx, WH_EARG, "logit probabilities: logits and probabilities of %d ids (rows %zu and %zu apart) are needed", vocab, ld, probs_ld);
  if (((uintptr_t)temperature | (uintptr_t)probs) % 4 || (uintptr_t)logits % (f16 ? 2 : 4))
    return wh_fail(ctx, WH_EARG, "logit probabilities: misaligned arrays");
  const size_t nodes = (size_t)t->batch * t->rows;
  if (nodes * PT >= (size_t)1 << 32) return wh_fail(ctx, WH_EARG, "logit probabilities: %zu rows in one call", nodes);
  const size_t in = f16 ? 2 : 4;
  if (rows_meet(logits, vocab * in, ld * in, probs, 4 * (size_t)vocab, 4 * probs_ld, nodes))
    return wh_fail(ctx, WH_EARG, "logit probabilities: they overlap the logits");
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "logit probabilities: %s", hipGetErrorString(e));
  const ProbsArgs a{logits, ld, probs, probs_ld, temperature, t->count, t->rows, vocab};
  ProfScope prof(ctx, "logit_probs", 0.0, (double)nodes * vocab * (in + 4));
  if (f16) wh_launch(ctx, probs_kernel<_Float16>, (unsigned)nodes, PT, 0, a);
  else wh_launch(ctx, probs_kernel<float>, (unsigned)nodes, PT, 0, a);
  return wh_launched(ctx, "logit probabilities");
}

int launch_tree_sample(wh_ctx *ctx, const wh_tree *t, const float *probs, const float *drafts, int vocab, size_t ld, const float *u, uint32_t *picks) {
  if (int rc = tree_check(ctx, "tree sample", t)) return rc;
  if (!probs || !u || !picks || (t->rows > 1 && !t->tokens) || vocab <= 0 || vocab > 1 << 28 || ld < (size_t)vocab)
    return wh_fail(ctx, WH_EARG, "tree sample: probabilities of %d ids (%zu apart), random numbers, picks, and the nodes' tokens are needed", vocab, ld);
  if (((uintptr_t)probs | (uintptr_t)drafts | (uintptr_t)u | (uintptr_t)picks) % 4) return wh_fail(ctx, WH_EARG, "tree sample: misaligned arrays");
  if ((size_t)t->batch * ST >= (size_t)1 << 32) return wh_fail(ctx, WH_EARG, "tree sample: %d sequences in one call", t->batch);
  const size_t nodes = (size_t)t->batch * t->rows;
  auto over = [&](const void *x, size_t values, size_t step) { return x && rows_meet(x, 4 * values, 4 * step, picks, 4 * nodes, 0, nodes); };
  if (over(probs, vocab, ld) || over(drafts, vocab, ld) || over(u, 1, 1) || over(t->tokens, 1, 1))
    return wh_fail(ctx, WH_EARG, "tree sample: the picks overlap what is read");
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "tree sample: %s", hipGetErrorString(e));
  const SampleArgs a{probs, drafts, u, t->count, t->tokens, t->mask, t->mask_stride, ld, t->rows, (t->rows + 31) / 32, vocab, picks};
  ProfScope prof(ctx, "tree_sample", 0.0, 4.0 * t->batch * vocab * (drafts ? 2 : 1));
  if (drafts) wh_launch(ctx, sample_kernel<true>, (unsigned)t->batch, ST, 0, a);
  else wh_launch(ctx, sample_kernel<false>, (unsigned)t->batch, ST, 0, a);
  return wh_launched(ctx, "tree sample");
}
