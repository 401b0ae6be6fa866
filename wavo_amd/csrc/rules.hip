// The requests' rules on rows of logits (include/wavo_hip.h, wh_logit_rules): penalties for ids that the
// text holds, biases, masks, the first maximum and its log-softmax.
//
// Bound by reading and writing the rows.  A workgroup takes 4096 ids of a sequence and several of its rows (nodes):
// what the sequence's text and biases say of an id is the same for all of them, so it is counted once, in LDS, and
// then kept in the registers of the thread that has the id (16 ids a thread).  Only ids among the tokens of the
// tree differ from node to node; a workgroup that has any counts them for every node again.  Otherwise its
// wavefronts go through the rows without meeting, each with the next row's loads under way, and leave a maximum and a
// sum of their own, which a second launch joins (one wavefront a row).
//
// The log-softmax is kept as the sum of exp(x − max) over every id but the maximum itself, so that a row
// with one likely id keeps its precision: logprob = −log1p(sum).
#include <algorithm>
#include <climits>

#include "internal.h"
#include "xlane.h"

namespace {

constexpr int RT = 256, PER = 16, IDS = PER * RT;  // threads, ids per thread and per workgroup
constexpr int NODES = TREE_ROWS;

struct RulePart {
  float best, rest;
  int at, pad;
};

struct RuleArgs {
  const int32_t *n, *count;
  const uint32_t *tokens, *mask;
  size_t mask_stride;
  int rows, words;
  const float *penalty;
  const uint32_t *history;
  int history_cols, from;
  const int32_t *bias_start;
  const uint32_t *bias_id;
  const float *bias;
  int bias_len;
  const uint32_t *allow;
  const void *logits;
  void *out;
  int vocab, chunks, group, groups;  // rows per workgroup; workgroups per sequence and chunk
  size_t ld;
  RulePart *part;  // [batch * rows][chunks][wavefront], or NULL: neither picks nor log-probabilities are asked for
};

__device__ __forceinline__ bool better(float ov, int oi, float v, int i) { return ov > v || (ov == v && oi < i); }

// x / r rounded once, for many x: from the reciprocal ri = 1 / r (rounded once), twice corrected by the remainder
// (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).  exact: r is
// where the remainders are numbers; quotients that are not are divided as they stand.
__device__ __forceinline__ float divide(float x, float r, float ri, bool exact) {
  float q = x * ri;
  if (!(exact && q > 0x1p-60f && q < 0x1p60f)) return x / r;
  q = __builtin_fmaf(__builtin_fmaf(-q, r, x), ri, q);
  return __builtin_fmaf(__builtin_fmaf(-q, r, x), ri, q);
}

// 16 bytes of a row of any alignment: 4 or 8 values.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
template <typename T>
struct Piece {
  typedef floatx4 type;
  typedef floatx4 any __attribute__((aligned(4)));
  static constexpr int N = 4;
};
template <>
struct Piece<_Float16> {
  typedef half8 type;
  typedef half8 any __attribute__((aligned(2)));
  static constexpr int N = 8;
};

template <typename T>
__global__ __launch_bounds__(RT) void rules_kernel(RuleArgs a) {
#pragma clang fp contract(off)  // the rules' sums and products are rounded one by one
  constexpr int V = Piece<T>::N, G = PER / V;  // ids per load, loads
  __shared__ uint32_t times[IDS];
  __shared__ int entry[IDS];
  __shared__ uint16_t who[NODES], what[NODES];  // the nodes whose tokens are among these ids
  __shared__ int whos;
  const int tid = threadIdx.x;
  const int chunk = blockIdx.x % a.chunks, rest_ = blockIdx.x / a.chunks, part_of = rest_ % a.groups, b = rest_ / a.groups;
  const int count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows;
  const int i0 = part_of * a.group, i1 = min(i0 + a.group, count);
  if (i0 >= i1) return;
  const int id0 = chunk * IDS;
  // This thread's ids: V from id0 + V * (tid + RT * t) on, t < G.
  const bool whole = id0 + IDS <= a.vocab;
  typedef typename Piece<T>::type P;
  P now[G];
  uint32_t ok[G];
  auto load = [&](int i) {
    const size_t row = (size_t)b * a.rows + i;
    const T *in = (const T *)a.logits + row * a.ld + id0;
    const uint32_t *allow = a.allow ? a.allow + row * ((a.vocab + 31) / 32) + id0 / 32 : nullptr;
#pragma unroll
    for (int t = 0; t < G; t++) {
      const int l = V * (tid + RT * t);
      if (whole) {
        now[t] = *(const typename Piece<T>::any *)(in + l);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) now[t][e] = id0 + l + e < a.vocab ? in[l + e] : (T)-INFINITY;
      }
      ok[t] = allow && (whole || id0 + l < a.vocab) ? allow[l / 32] >> (l % 32) : 0xffffffffu;
    }
  };
  load(i0);

  // How often each id stands in the sequence's text, and its bias entry.
  const bool counted = a.penalty != nullptr, biased = a.bias_start != nullptr;
  float fc[PER], bias[PER], r = 1.0f, ri = 1.0f, f = 0.0f, p = 0.0f;
  uint32_t hit = 0;
#pragma unroll
  for (int e = 0; e < PER; e++) fc[e] = 0.0f, bias[e] = 0.0f;
  auto look = [&] {  // the counts of this thread's ids
    hit = 0;
#pragma unroll
    for (int t = 0; t < G; t++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        const uint32_t c = times[V * (tid + RT * t) + e];
        fc[V * t + e] = f * (float)c;
        hit |= (c ? 1u : 0u) << (V * t + e);
      }
  };
  int listed = 0;
  if (counted || biased) {
    for (int x = tid; x < IDS; x += RT) times[x] = 0, entry[x] = -1;
    if (tid == 0) whos = 0;
    __syncthreads();
    if (counted) {
      r = a.penalty[3 * b], f = a.penalty[3 * b + 1], p = a.penalty[3 * b + 2];
      ri = 1.0f / r;
      const int n = a.history ? min(max(a.n[b], 0), a.history_cols) : 0;
      const uint32_t *text = a.history + (size_t)b * a.history_cols;
      for (int x = a.from + tid; x < n; x += 8 * RT) {  // (8 ids' loads at a time)
        uint32_t id[8];
#pragma unroll
        for (int y = 0; y < 8; y++) id[y] = text[min(x + RT * y, n - 1)] - (uint32_t)id0;
#pragma unroll
        for (int y = 0; y < 8; y++)
          if (x + RT * y < n && id[y] < (uint32_t)IDS) atomicAdd(&times[id[y]], 1u);
      }
      if (a.mask)
        for (int j = tid; j < count; j += RT) {
          const uint32_t id = a.tokens[(size_t)b * a.rows + j] - (uint32_t)id0;
          if (id < (uint32_t)IDS) {
            const int at = atomicAdd(&whos, 1);
            who[at] = (uint16_t)j, what[at] = (uint16_t)id;
          }
        }
    }
    if (biased) {
      const int e0 = max(a.bias_start[b], 0), e1 = min(a.bias_start[b + 1], a.bias_len);
      for (int x = e0 + tid; x < e1; x += RT) {
        const uint32_t id = a.bias_id[x] - (uint32_t)id0;
        if (id < (uint32_t)IDS) atomicMax(&entry[id], x);
      }
    }
    __syncthreads();
    listed = whos;
    if (biased)
#pragma unroll
      for (int t = 0; t < G; t++)
#pragma unroll
        for (int e = 0; e < V; e++) {
          const int at = entry[V * (tid + RT * t) + e];
          if (at >= 0) bias[V * t + e] = a.bias[at];
        }
    if (counted && !listed) look();
  }
  const bool exact = r > 0x1p-30f && r < 0x1p30f;

  for (int i = i0; i < i1; i++) {
    if (listed) {  // (every wavefront's: the tokens of the nodes that node i sees)
      const uint32_t *mask = a.mask + (size_t)b * a.mask_stride + (size_t)i * a.words;
      __syncthreads();
      for (int x = tid; x < listed; x += RT)
        if (mask[who[x] / 32] >> (who[x] % 32) & 1) atomicAdd(&times[what[x]], 1u);
      __syncthreads();
      look();
      __syncthreads();
      for (int x = tid; x < listed; x += RT)
        if (mask[who[x] / 32] >> (who[x] % 32) & 1) atomicAdd(&times[what[x]], 0xffffffffu);
    }
    float v[PER];
#pragma unroll
    for (int t = 0; t < G; t++)
#pragma unroll
      for (int e = 0; e < V; e++) v[V * t + e] = (float)now[t][e];
    uint32_t allowed[G];
#pragma unroll
    for (int t = 0; t < G; t++) allowed[t] = ok[t];
    if (i + 1 < i1) load(i + 1);
    const size_t row = (size_t)b * a.rows + i;
    T *out = a.out ? (T *)a.out + row * a.ld + id0 : nullptr;
#pragma unroll
    for (int t = 0; t < G; t++) {
      if (counted && __any((hit >> (V * t) & ((1u << V) - 1u)) != 0))
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float x = v[V * t + e], y = x > 0.0f ? divide(x, r, ri, exact) : x * r;
          if (hit >> (V * t + e) & 1) v[V * t + e] = (y - fc[V * t + e]) - p;
        }
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float x = v[V * t + e] + bias[V * t + e];
        v[V * t + e] = allowed[t] >> e & 1 ? x : -INFINITY;
      }
    }
    if (out)
#pragma unroll
      for (int t = 0; t < G; t++) {
        const int l = V * (tid + RT * t);
        P w;
#pragma unroll
        for (int e = 0; e < V; e++) w[e] = (T)v[V * t + e];
        if (whole) {
          *(typename Piece<T>::any *)(out + l) = w;
        } else {
#pragma unroll
          for (int e = 0; e < V; e++)
            if (id0 + l + e < a.vocab) out[l + e] = w[e];
        }
      }
    if (!a.part) continue;
    float best = -INFINITY;
#pragma unroll
    for (int e = 0; e < PER; e++) best = fmaxf(best, v[e]);
    best = xlane::wave_max(best);
    // Its first place (ids that are not there hold −∞, as masked ones do), and the others' mass against it.
    int at = INT_MAX;
    if (best > -INFINITY)
#pragma unroll
      for (int e = PER - 1; e >= 0; e--)
        if (v[e] == best) at = V * (tid + RT * (e / V)) + e % V;
    for (int d = 32; d; d >>= 1) at = min(at, __shfl_xor(at, d));
    float rest = 0.0f;
    const float m = best == -INFINITY ? 0.0f : best;
#pragma unroll
    for (int e = 0; e < PER; e++)
      if (V * (tid + RT * (e / V)) + e % V != at) rest += __expf(v[e] - m);
    rest = xlane::wave_sum(rest);
    if ((tid & 63) == 0) a.part[(row * a.chunks + chunk) * (RT / 64) + tid / 64] = {best, rest, at == INT_MAX ? at : id0 + at, 0};
  }
}

// (best, rest, at) of two runs of ids: the greater maximum, and the other one's mass against it.
__device__ __forceinline__ void join(float &best, float &rest, int &at, float ob, float orest, int oat) {
  if (better(ob, oat, best, at)) {
    float x = best;
    best = ob, ob = x;
    x = rest, rest = orest, orest = x;
    const int y = at;
    at = oat, oat = y;
  }
  if (ob == -INFINITY) rest += orest;  // (nothing there, or NaN)
  else rest += (1.0f + orest) * __expf(ob - best);
}

// One wave per row joins its parts.
__global__ __launch_bounds__(64) void rules_pick_kernel(const RulePart *part, const int32_t *counts, int rows, int parts,
                                                        uint32_t *pick, float *logprob) {
  const int row = blockIdx.x, lane = threadIdx.x;
  if (counts && row % rows >= counts[row / rows]) return;
  float best = -INFINITY, rest = 0.0f;
  int at = INT_MAX;
  for (int c = lane; c < parts; c += 256) {  // (4 loads at a time)
    RulePart p[4];
#pragma unroll
    for (int y = 0; y < 4; y++) p[y] = part[(size_t)row * parts + min(c + 64 * y, parts - 1)];
#pragma unroll
    for (int y = 0; y < 4; y++)
      if (c + 64 * y < parts) join(best, rest, at, p[y].best, p[y].rest, p[y].at);
  }
  for (int d = 32; d; d >>= 1) {
    const float ob = __shfl_xor(best, d), orest = __shfl_xor(rest, d);
    const int oat = __shfl_xor(at, d);
    join(best, rest, at, ob, orest, oat);
  }
  if (lane) return;
  if (pick) pick[row] = best == -INFINITY ? 0xffffffffu : (uint32_t)at;
  // (best − best: NaN beside an infinity, as in the quotient it stands for)
  if (logprob) logprob[row] = rest != rest ? rest : best == -INFINITY ? best : (best - best) - log1pf(rest);
}

}  // namespace

int launch_logit_rules(wh_ctx *ctx, const wh_tree *t, const wh_rules *r, const void *logits, void *out, int vocab, size_t ld,
                       int f16, uint32_t *pick, float *logprob) {
  if (int rc = tree_check(ctx, "logit rules", t)) return rc;
  if (!r || !logits || (!out && !pick && !logprob) || vocab <= 0 || vocab > 1 << 28 || ld < (size_t)vocab)
    return wh_fail(ctx, WH_EARG, "logit rules: rules, logits, an output and rows of %d ids (%zu apart) are needed", vocab, ld);
  if (r->history && (r->history_cols <= 0 || r->from < 0))
    return wh_fail(ctx, WH_EARG, "logit rules: texts of %d ids from %d on", r->history_cols, r->from);
  if (r->bias_start && (!r->bias_id || !r->bias || r->bias_len < 0))
    return wh_fail(ctx, WH_EARG, "logit rules: biases need their ids, values and number");
  if (r->penalty && t->mask && !t->tokens) return wh_fail(ctx, WH_EARG, "logit rules: the nodes' tokens are needed");
  if (((uintptr_t)r->penalty | (uintptr_t)r->history | (uintptr_t)r->bias_start | (uintptr_t)r->bias_id | (uintptr_t)r->bias |
       (uintptr_t)r->allow | (uintptr_t)pick | (uintptr_t)logprob) % 4 || ((uintptr_t)logits | (uintptr_t)out) % (f16 ? 2 : 4))
    return wh_fail(ctx, WH_EARG, "logit rules: misaligned arrays");
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "logit rules: %s", hipGetErrorString(e));
  const size_t nodes = (size_t)t->batch * t->rows;
  const int chunks = (vocab + IDS - 1) / IDS, parts = chunks * (RT / 64);
  // Rows per workgroup: all of a sequence's, or as many as leave 4 workgroups a CU.
  const size_t want = 4 * (size_t)(ctx->cus > 0 ? ctx->cus : 256), each = (size_t)chunks * t->batch;
  int groups = (int)std::min<size_t>(t->rows, (want + each - 1) / each);
  const int group = (t->rows + groups - 1) / groups;
  groups = (t->rows + group - 1) / group;
  if (each * groups >= (size_t)1 << 24) return wh_fail(ctx, WH_EARG, "logit rules: %zu rows of %d ids", nodes, vocab);
  RulePart *part = nullptr;
  if ((pick || logprob) && !(part = (RulePart *)wh_scratch(ctx, sizeof(RulePart) * parts * nodes))) return WH_EOOM;
  const RuleArgs a{t->n, t->count, t->tokens, t->mask, t->mask_stride, t->rows, (t->rows + 31) / 32, r->penalty, r->history,
                   r->history_cols, r->from, r->bias_start, r->bias_id, r->bias, r->bias_len, r->allow, logits, out, vocab,
                   chunks, group, groups, ld, part};
  {
    ProfScope prof(ctx, "logit_rules", 0.0, (double)nodes * vocab * (f16 ? 2 : 4) * (out ? 2 : 1));
    if (f16) wh_launch(ctx, rules_kernel<_Float16>, (int)each * groups, RT, 0, a);
    else wh_launch(ctx, rules_kernel<float>, (int)each * groups, RT, 0, a);
    if (int rc = wh_launched(ctx, "logit rules")) return rc;
  }
  if (!part) return WH_OK;
  ProfScope prof(ctx, "logit_pick", 0.0, (double)sizeof(RulePart) * parts * nodes);
  wh_launch(ctx, rules_pick_kernel, (int)nodes, 64, 0, (const RulePart *)part, t->count, t->rows, parts, pick, logprob);
  return wh_launched(ctx, "logit pick");
}
