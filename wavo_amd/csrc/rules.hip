// The requests' rules on rows of logits (include/wavo_hip.h, wh_logit_rules): penalties for ids that the
// text holds, biases, masks, the first maximum and its log-softmax.
//
// The log-softmax is kept as the sum of exp(x − max) over every id but the maximum itself, so that a row
// with one likely id keeps its precision: logprob = −log1p(sum).
#include <algorithm>
#include <climits>

#include "internal.h"
#include "xlane.h"

namespace {

constexpr int RT = 256, RQ = 4, IDS = 4 * RT * RQ;  // threads, groups of 4 ids per thread, ids per workgroup

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
  int vocab, chunks;
  size_t ld;
  RulePart *part;  // [batch * rows][chunks], or NULL: neither picks nor log-probabilities are asked for
};

__device__ __forceinline__ bool better(float ov, int oi, float v, int i) { return ov > v || (ov == v && oi < i); }

// One workgroup per row and 4096 ids: how often each of them stands in the text and which bias entry it has,
// counted in LDS, then the ids' values.
template <typename T>
__global__ __launch_bounds__(RT) void rules_kernel(RuleArgs a) {
#pragma clang fp contract(off)  // the rules' sums and products are rounded one by one
  __shared__ uint32_t times[IDS];
  __shared__ int entry[IDS];
  __shared__ float redv[4], reds[4];
  __shared__ int redi[4];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, b = row / a.rows, i = row % a.rows;
  const int count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows;
  if (i >= count) return;
  const int id0 = chunk * IDS;
  for (int x = tid; x < IDS; x += RT) times[x] = 0, entry[x] = -1;
  __syncthreads();
  if (a.penalty) {
    const int n = a.history ? min(max(a.n[b], 0), a.history_cols) : 0;
    for (int x = a.from + tid; x < n; x += RT) {
      const uint32_t id = a.history[(size_t)b * a.history_cols + x] - (uint32_t)id0;
      if (id < (uint32_t)IDS) atomicAdd(&times[id], 1u);
    }
    if (a.mask)
      for (int j = tid; j < count; j += RT) {
        const uint32_t id = a.tokens[(size_t)b * a.rows + j] - (uint32_t)id0;
        if (id < (uint32_t)IDS && (a.mask[(size_t)b * a.mask_stride + (size_t)i * a.words + j / 32] >> (j % 32) & 1))
          atomicAdd(&times[id], 1u);
      }
  }
  if (a.bias_start) {
    const int e0 = max(a.bias_start[b], 0), e1 = min(a.bias_start[b + 1], a.bias_len);
    for (int x = e0 + tid; x < e1; x += RT) {
      const uint32_t id = a.bias_id[x] - (uint32_t)id0;
      if (id < (uint32_t)IDS) atomicMax(&entry[id], x);
    }
  }
  __syncthreads();
  const float r = a.penalty ? a.penalty[3 * b] : 1.0f, f = a.penalty ? a.penalty[3 * b + 1] : 0.0f,
              p = a.penalty ? a.penalty[3 * b + 2] : 0.0f;
  const T *in = (const T *)a.logits + (size_t)row * a.ld;
  T *out = a.out ? (T *)a.out + (size_t)row * a.ld : nullptr;
  const uint32_t *allow = a.allow ? a.allow + (size_t)row * ((a.vocab + 31) / 32) : nullptr;
  float v[4 * RQ];
  float best = -INFINITY;
  int at = INT_MAX;
#pragma unroll
  for (int t = 0; t < RQ; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int l = 4 * (tid + RT * t) + e, id = id0 + l;
      float x = -INFINITY;
      if (id < a.vocab) {
        x = (float)in[id];
        const float c = (float)times[l];
        if (times[l]) x = ((x > 0.0f ? x / r : x * r) - f * c) - p;
        if (entry[l] >= 0) x = x + a.bias[entry[l]];
        if (allow && !(allow[id / 32] >> (id % 32) & 1)) x = -INFINITY;
        if (out) out[id] = (T)x;
      }
      v[4 * t + e] = x;
      if (x > best) best = x, at = id;
    }
  if (!a.part) return;
  xlane::wave_first_max(best, at, better);
  if ((tid & 63) == 0) redv[wave] = best, redi[wave] = at;
  __syncthreads();
  best = redv[0], at = redi[0];
  for (int w = 1; w < 4; w++)
    if (better(redv[w], redi[w], best, at)) best = redv[w], at = redi[w];
  float rest = 0.0f;
  const float m = best == -INFINITY ? 0.0f : best;
#pragma unroll
  for (int t = 0; t < RQ; t++)
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (id0 + 4 * (tid + RT * t) + e != at) rest += __expf(v[4 * t + e] - m);
  rest = xlane::wave_sum(rest);
  if ((tid & 63) == 0) reds[wave] = rest;
  __syncthreads();
  if (tid == 0) a.part[(size_t)row * a.chunks + chunk] = {best, reds[0] + reds[1] + reds[2] + reds[3], at, 0};
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

// One wave per row joins its chunks.
__global__ __launch_bounds__(64) void rules_pick_kernel(const RulePart *part, const int32_t *counts, int rows, int chunks,
                                                        uint32_t *pick, float *logprob) {
  const int row = blockIdx.x, lane = threadIdx.x;
  if (counts && row % rows >= counts[row / rows]) return;
  float best = -INFINITY, rest = 0.0f;
  int at = INT_MAX;
  for (int c = lane; c < chunks; c += 64) {
    const RulePart p = part[(size_t)row * chunks + c];
    join(best, rest, at, p.best, p.rest, p.at);
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
  const int chunks = (vocab + IDS - 1) / IDS, nodes = t->batch * t->rows;
  if ((size_t)chunks * nodes > INT_MAX) return wh_fail(ctx, WH_EARG, "logit rules: %d rows of %d ids", nodes, vocab);
  RulePart *part = nullptr;
  if ((pick || logprob) && !(part = (RulePart *)wh_scratch(ctx, sizeof(RulePart) * (size_t)chunks * nodes))) return WH_EOOM;
  const RuleArgs a{t->n, t->count, t->tokens, t->mask, t->mask_stride, t->rows, (t->rows + 31) / 32, r->penalty, r->history,
                   r->history_cols, r->from, r->bias_start, r->bias_id, r->bias, r->bias_len, r->allow, logits, out, vocab,
                   chunks, ld, part};
  {
    ProfScope prof(ctx, "logit_rules", 0.0, (double)nodes * vocab * (f16 ? 2 : 4) * (out ? 2 : 1));
    if (f16) wh_launch(ctx, rules_kernel<_Float16>, chunks * nodes, RT, 0, a);
    else wh_launch(ctx, rules_kernel<float>, chunks * nodes, RT, 0, a);
    if (int rc = wh_launched(ctx, "logit rules")) return rc;
  }
  if (!part) return WH_OK;
  ProfScope prof(ctx, "logit_pick", 0.0, (double)sizeof(RulePart) * chunks * nodes);
  wh_launch(ctx, rules_pick_kernel, nodes, 64, 0, (const RulePart *)part, t->count, t->rows, chunks, pick, logprob);
  return wh_launched(ctx, "logit pick");
}
