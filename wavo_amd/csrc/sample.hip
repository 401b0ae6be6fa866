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

// One row per workgroup: its maximum and the sum of exp((x - max) / T) in one pass, the probabilities in a second one.
template <typename T>
__global__ __launch_bounds__(PT) void probs_kernel(ProbsArgs a) {
  __shared__ float tops[PT / 64], sums[PT / 64];
  __shared__ int first;
  const int row = blockIdx.x, b = row / a.rows, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  if (a.count && row - b * a.rows >= a.count[b]) return;
  const T *x = (const T *)a.logits + (size_t)row * a.ld;
  float *y = a.probs + (size_t)row * a.probs_ld;
  const float t = a.temperature ? a.temperature[b] : 1.0f;
  float top = -INFINITY;
  for (int i = tid; i < a.vocab; i += PT) top = fmaxf(top, (float)x[i]);
  top = xlane::wave_max(top);
  if (lane == 0) tops[wave] = top;
  if (tid == 0) first = INT_MAX;
  __syncthreads();
  top = tops[lane % (PT / 64)];
  top = xlane::wave_max(top);
  if (!(t > 0.0f)) {  // all of it to the first maximum
    int at = INT_MAX;
    for (int i = tid; i < a.vocab && at == INT_MAX; i += PT)
      if ((float)x[i] == top && top > -INFINITY) at = i;
    if (at != INT_MAX) atomicMin(&first, at);
    __syncthreads();
    for (int i = tid; i < a.vocab; i += PT) y[i] = i == first ? 1.0f : 0.0f;
    return;
  }
  const float base = top == -INFINITY ? 0.0f : top, k = fminf(1.44269504088896341f / t, 3.402823466e38f);
  float sum = 0.0f;
  for (int i = tid; i < a.vocab; i += PT) sum += __builtin_amdgcn_exp2f(((float)x[i] - base) * k);
  sum = xlane::wave_sum(sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  sum = lane < PT / 64 ? sums[lane] : 0.0f;
  sum = xlane::wave_sum(sum);
  const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int i = tid; i < a.vocab; i += PT) y[i] = __builtin_amdgcn_exp2f(((float)x[i] - base) * k) * scale;
}

struct SampleArgs {
  const float *p, *q, *u;
  const int32_t *count;
  const uint32_t *tokens, *mask;
  size_t mask_stride, ld;
  int rows, words, vocab;
  uint32_t *picks;
};

constexpr int ST = 1024;  // threads of a sequence's workgroup

// The sum over the workgroup, the same for every thread; `part` is free again after the next barrier.
__device__ __forceinline__ double block_sum(double v, double *part) {
  v = xlane::wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < ST / 64; i++) s += part[i];
  return s;
}

// A sequence's walk by one workgroup.  What is left of a node's probabilities after rejections of its children's tokens is
// made anew from p and q whenever it is read: with drafts, w = max(0, w / Z - q) round by round; without, zero at the tokens.
__global__ __launch_bounds__(ST) void sample_kernel(SampleArgs a) {
  __shared__ double part[ST / 64], inverse[TREE_ROWS];
  __shared__ uint32_t out[TREE_ROWS];
  __shared__ int found;
  const int b = blockIdx.x, tid = threadIdx.x, count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows;
  if (count == 0) return;
  const size_t row0 = (size_t)b * a.rows;
  const uint32_t *tokens = a.tokens + row0, *mask = a.mask ? a.mask + (size_t)b * a.mask_stride : nullptr;
  for (int i = tid; i < count; i += ST) out[i] = NONE;
  if (tid == 0) found = -1;
  int at = 0, rounds = 0;  // the node, and how many of its children were rejected
  double total = 1.0;
  const float *p = a.p + row0 * a.ld, *q = a.q ? a.q + row0 * a.ld : nullptr;
  // (without drafts: the tokens that are out, in `inverse` as numbers)
  auto left = [&](int x) {
    double w = p[x];
    if (q) {
      const double y = q[x];
      for (int r = 0; r < rounds; r++) w = fmax(w * inverse[r] - y, 0.0);
    } else {
      for (int r = 0; r < rounds; r++) w = inverse[r] == (double)x ? 0.0 : w;
    }
    return w;
  };
  __syncthreads();
  for (int i = 1; i < count; i++) {
    // i's parent: the highest node below it that it sees.
    int parent = mask ? -1 : i - 1;
    if (mask) {
      const uint32_t *m = mask + (size_t)i * a.words;
      for (int w = (i - 1) / 32; w >= 0 && parent < 0; w--) {
        const uint32_t bits = m[w] & (w == i / 32 ? (1u << i % 32) - 1u : 0xffffffffu);
        if (bits) parent = 32 * w + 31 - __clz(bits);
      }
    }
    if (parent != at || !(total > 0.0)) continue;
    const uint32_t x = tokens[i];
    const double mine = x < (uint32_t)a.vocab ? left((int)x) : 0.0, u = a.u[row0 + i];
    if (x < (uint32_t)a.vocab && u * (q ? (double)q[x] : 1.0) * total < mine) {
      if (tid == 0) out[at] = x;
      at = i, rounds = 0, total = 1.0;
      p = a.p + (row0 + i) * a.ld, q = a.q ? a.q + (row0 + i) * a.ld : nullptr;
      continue;
    }
    if (x >= (uint32_t)a.vocab) continue;  // (no draft of this vocabulary)
    __syncthreads();
    if (tid == 0) inverse[rounds] = q ? 1.0 / total : (double)x;
    __syncthreads();
    rounds++;
    if (q) {
      double sum = 0.0;
      for (int y = tid; y < a.vocab; y += ST) sum += left(y);
      total = block_sum(sum, part);
    } else {
      total -= mine;
    }
  }
  // The draw: each wavefront sums a run of ids, the one that holds the place looks for it.
  constexpr int WV = ST / 64;
  const int wave = tid >> 6, lane = tid & 63, run = ((a.vocab + WV - 1) / WV + 63) / 64 * 64;
  for (int attempt = 0; attempt < 2; attempt++) {
    const int begin = min(wave * run, a.vocab), end = min(begin + run, a.vocab);
    double sum = 0.0;
    for (int x = begin + lane; x < end; x += 64) sum += left(x);
    sum = xlane::wave_sum(sum);
    __syncthreads();
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    double all = 0.0, before = 0.0;
    for (int i = 0; i < WV; i++) {
      if (i == wave) before = all;
      all += part[i];
    }
    if (!(all > 0.0)) {  // nothing left: from the node's probabilities themselves
      rounds = 0;
      continue;
    }
    const double place = (double)a.u[row0] * all;
    // One run holds the place.  (Its own running sums may end a last bit before it: then it is at the run's last id.)
    if (before <= place && place < before + part[wave]) {
      int last = -1, hit = -1;
      for (int x0 = begin; x0 < end && hit < 0; x0 += 64) {
        const int x = x0 + lane;
        const double w = x < end ? left(x) : 0.0;
        double c = w;  // running sums of the 64
        for (int d = 1; d < 64; d *= 2) {
          const double o = __shfl_up(c, d);
          if (lane >= d) c += o;
        }
        const uint64_t over = __ballot(w > 0.0 && before + c > place), some = __ballot(w > 0.0);
        if (some) last = x0 + 63 - __clzll(some);
        if (over) hit = x0 + (int)__builtin_ctzll(over);
        before += __shfl(c, 63);
      }
      if (lane == 0) found = hit >= 0 ? hit : last;
    }
    __syncthreads();
    if (found < 0) {  // (a random number that is not below one: the last id of any mass)
      int most = -1;
      for (int x = tid; x < a.vocab; x += ST)
        if (left(x) > 0.0) most = x;
      atomicMax(&found, most);
      __syncthreads();
    }
    if (tid == 0) out[at] = (uint32_t)found;
    break;
  }
  __syncthreads();
  for (int i = tid; i < count; i += ST) a.picks[row0 + i] = out[i];
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
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "logit probabilities: %s", hipGetErrorString(e));
  const ProbsArgs a{logits, ld, probs, probs_ld, temperature, t->count, t->rows, vocab};
  ProfScope prof(ctx, "logit_probs", 0.0, (double)nodes * vocab * (f16 ? 6 : 8));
  if (f16) wh_launch(ctx, probs_kernel<_Float16>, (unsigned)nodes, PT, 0, a);
  else wh_launch(ctx, probs_kernel<float>, (unsigned)nodes, PT, 0, a);
  return wh_launched(ctx, "logit probabilities");
}

int launch_tree_sample(wh_ctx *ctx, const wh_tree *t, const float *probs, const float *drafts, int vocab, size_t ld, const float *u, uint32_t *picks) {
  if (int rc = tree_check(ctx, "tree sample", t)) return rc;
  if (!probs || !u || !picks || (t->rows > 1 && !t->tokens) || vocab <= 0 || vocab > 1 << 28 || ld < (size_t)vocab)
    return wh_fail(ctx, WH_EARG, "tree sample: probabilities of %d ids (%zu apart), random numbers, picks, and the nodes' tokens are needed", vocab, ld);
  if (((uintptr_t)probs | (uintptr_t)drafts | (uintptr_t)u | (uintptr_t)picks) % 4) return wh_fail(ctx, WH_EARG, "tree sample: misaligned arrays");
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "tree sample: %s", hipGetErrorString(e));
  const SampleArgs a{probs, drafts, u, t->count, t->tokens, t->mask, t->mask_stride, ld, t->rows, (t->rows + 31) / 32, vocab, picks};
  ProfScope prof(ctx, "tree_sample", 0.0, 4.0 * t->batch * vocab * (drafts ? 2 : 1));
  wh_launch(ctx, sample_kernel, (unsigned)t->batch, ST, 0, a);
  return wh_launched(ctx, "tree sample");
}
