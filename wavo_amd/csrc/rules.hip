// The requests' rules on rows of logits (include/wavo_hip.h, wh_logit_rules): penalties for ids that the
// text holds, biases, masks, the first maximum and its log-softmax.
//
// A workgroup takes 2048 ids of a sequence and several of its rows (nodes).  What the sequence's text and biases say of
// an id is the same for all of them: it is counted once, in LDS, and each wavefront lists those of its 512 ids that a
// rule can change (few, but for the most frequent ids).  Then the wavefronts go through the rows without meeting, two
// rows' loads ahead: a row's values go to LDS, the listed ones are changed there, a lane for each, and come back.  The
// tree's tokens differ from node to node: those on a node's path are added to the counts before its row and taken
// back after it.  Each wavefront leaves a maximum and a sum of its own, which the last workgroup of a run of rows to
// be through joins, or a second launch (one wavefront a row).
//
// The log-softmax is kept as the sum of exp(x − max) over every id but the maximum itself, so that a row
// with one likely id keeps its precision: logprob = −log1p(sum).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "internal.h"
#include "xlane.h"

namespace {

constexpr int RT = 256, PER = 8, IDS = PER * RT, WIDS = 64 * PER;  // threads; ids per thread, workgroup and wavefront
constexpr int GROUP = 10, WORDS = TREE_ROWS / 64;  // rows of a workgroup, at most; 64-bit words of a node's path

struct RulePart {
  float best, rest;
  int at, pad;
};
// For parts that pass between workgroups of one launch: each half is stored to and loaded from where all XCDs see it.
__device__ __forceinline__ void store_part(RulePart *p, RulePart x) {
  const uint64_t *w = (const uint64_t *)&x;
  for (int e = 0; e < 2; e++) __hip_atomic_store((uint64_t *)p + e, w[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ RulePart load_part(const RulePart *p) {
  RulePart x;
  for (int e = 0; e < 2; e++)
    ((uint64_t *)&x)[e] = __hip_atomic_load((const uint64_t *)p + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return x;
}

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
  uint32_t *pick;
  float *logprob;
  int *done;  // [batch * groups] workgroups that are through (0 between launches), or NULL: another launch joins the parts
};

__device__ __forceinline__ bool better(float ov, int oi, float v, int i) { return ov > v || (ov == v && oi < i); }

// 16 bytes of a row of any alignment: 4 or 8 values.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
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

// One wavefront joins a row's parts.
__device__ __forceinline__ void join_row(const RulePart *part, int parts, int lane, uint32_t *pick, float *logprob) {
  float best = -INFINITY, rest = 0.0f;
  int at = INT_MAX;
  for (int c = lane; c < parts; c += 256) {  // (4 loads at a time)
    RulePart p[4];
#pragma unroll
    for (int y = 0; y < 4; y++) p[y] = load_part(part + min(c + 64 * y, parts - 1));
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
  if (pick) *pick = best == -INFINITY ? 0xffffffffu : (uint32_t)at;
  // (best − best: NaN beside an infinity, as in the quotient it stands for)
  if (logprob) *logprob = rest != rest ? rest : best == -INFINITY ? best : (best - best) - log1pf(rest);
}

// Keeps what a wavefront does in LDS in the order it is written in (its accesses are served in order).
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }

// ALLOW, OUT, whole: what a row's pass loads and stores has to be the same for every row, so that a wait for one row's
// loads is not one for the next rows'.  61 rows of 131071 f16 ids for 8 requests, 16000 ids of text and 1000 biases
// each: 91 us (2.2 TB/s; 97 where the stores stay in L2); 24 rows of 51866 f32 ids for 16 requests: 33 us (3.7 TB/s; 40).
// A copy of the former rows in the same form takes 42 us; the rest is each row's chain of LDS trips, cross-lane sums and 232
// vector instructions, in as many wavefronts as LDS has room for (five workgroups a CU; 95 us with four).
template <typename T, bool ALLOW, bool OUT>
__global__ __launch_bounds__(RT, 5) void rules_kernel(RuleArgs a) {
#pragma clang fp contract(off)  // the rules' sums and products are rounded one by one
  constexpr int V = Piece<T>::N, G = PER / V;  // ids per load, loads
  typedef typename Piece<T>::type P;
  // times: twice an id's count, and 1 where a node has it as its token.  bias: the entry, then its value.  list: the ids of
  // each wavefront that a rule can change.  who: the nodes whose tokens are among these ids, then those tokens.
  __shared__ uint32_t times[IDS];
  __shared__ float bias[IDS];
  __shared__ __attribute__((aligned(16))) float values[IDS];
  __shared__ uint16_t list[IDS], who[TREE_ROWS];
  __shared__ uint64_t paths[GROUP][WORDS];  // per row of this workgroup: which nodes of `who` it sees
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunk = blockIdx.x % a.chunks, of = blockIdx.x / a.chunks, b = of / a.groups;
  const int i0 = (of - b * a.groups) * a.group, id0 = chunk * IDS;
  // This thread's ids: V from id0 + first + V * RT * t on, t < G.
  const int first = V * tid;
  auto mine = [&](int e) { return first + V * RT * (e / V) + e % V; };
  struct Row {
    P x[G];
    uint32_t ok[G];  // from bit 0 on, a bit per id
  };
  const size_t row0 = (size_t)b * a.rows;
  const bool whole = id0 + IDS <= a.vocab;
  auto load = [&](auto all, Row &w, int i) {
    const T *in = (const T *)a.logits + (row0 + i) * a.ld + id0;
    const uint32_t *allow = ALLOW ? a.allow + (row0 + i) * ((a.vocab + 31) / 32) + id0 / 32 : nullptr;
#pragma unroll
    for (int t = 0; t < G; t++) {
      const int l = first + V * RT * t, left = a.vocab - id0 - l;
      if constexpr (all) {
        w.x[t] = *(const typename Piece<T>::any *)(in + l);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) w.x[t][e] = e < left ? in[l + e] : (T)-INFINITY;
      }
      if constexpr (ALLOW) w.ok[t] = all || left > 0 ? allow[l / 32] >> (l % 32) : 0u;
    }
  };
  Row even, odd;  // rows i0, i0 + 2, .. and the others: each loaded again as soon as its values are in use
  auto load_first = [&](int last) {
    if (whole) load(std::true_type{}, even, i0), load(std::true_type{}, odd, min(i0 + 1, last));
    else load(std::false_type{}, even, i0), load(std::false_type{}, odd, min(i0 + 1, last));
  };
  // What is asked for before the sequence's numbers are known: its first rows and the text's first EARLY ids a thread (61
  // rows of 131071 ids for 8 requests 91.5 us, 93 asked for afterwards, 48 requests' one row of 51866 13.3 and 13.6; one
  // request's row 8.5 us of kernel either way).
  constexpr int EARLY = 2;
  const bool counted = a.penalty != nullptr, biased = a.bias_start != nullptr, has_text = counted && a.history;
  const uint32_t *text = has_text ? a.history + (size_t)b * a.history_cols : nullptr;
  uint32_t early[EARLY];
  if (has_text)
#pragma unroll
    for (int y = 0; y < EARLY; y++) early[y] = text[min(min(a.from, a.history_cols - 1) + RT * y + tid, a.history_cols - 1)];
  if (i0 == 0) load_first(a.rows - 1);
  const int count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows, i1 = min(i0 + a.group, count);
  const int n = has_text ? min(max(a.n[b], 0), a.history_cols) : 0;
  const float r = counted ? a.penalty[3 * b] : 1.0f, f = counted ? a.penalty[3 * b + 1] : 0.0f, p = counted ? a.penalty[3 * b + 2] : 0.0f;
  const int e0 = biased ? max(a.bias_start[b], 0) : 0, e1 = biased ? min(a.bias_start[b + 1], a.bias_len) : 0;
  if (i0 >= i1) return;
  if (i0) load_first(i1 - 1);

  int changes = 0, listed = 0;  // of this wavefront's list; of `who`
  int one = 0, token = -1;      // the lane's id on the list; its token of `who`, if it is this wavefront's
  float onebias = 0.0f;
  const int span = min(IDS, a.vocab - id0);
  if (counted || biased) {
    int *entry = (int *)bias, &whos = *(int *)values;
#pragma unroll
    for (int e = 0; e < PER; e++) times[tid + RT * e] = 0, entry[tid + RT * e] = -1;
    if (tid == 0) whos = 0;
    __syncthreads();
    if (counted) {
      auto add = [&](uint32_t id) {
        id -= (uint32_t)id0;
        if (id < (uint32_t)span) atomicAdd(&times[id], 2u);
      };
#pragma unroll
      for (int y = 0; y < EARLY; y++)
        if (a.from < n && a.from + RT * y + tid < n) add(early[y]);
      int x = a.from < n ? a.from + EARLY * RT : n;
      for (; x + 16 * RT <= n; x += 16 * RT) {  // (16 ids a thread at a time)
        u32x4 id[4];
#pragma unroll
        for (int y = 0; y < 4; y++) id[y] = *(const u32x4_a4 *)(text + x + 4 * (tid + RT * y));
#pragma unroll
        for (int y = 0; y < 16; y++) add(id[y / 4][y % 4]);
      }
      if (x < n) {
        uint32_t id[16];
#pragma unroll
        for (int y = 0; y < 16; y++) id[y] = text[min(x + RT * y + tid, n - 1)];
#pragma unroll
        for (int y = 0; y < 16; y++)
          if (x + RT * y + tid < n) add(id[y]);
      }
      if (a.mask)
        for (int j = tid; j < count; j += RT) {
          const uint32_t id = a.tokens[(size_t)b * a.rows + j] - (uint32_t)id0;
          if (id < (uint32_t)span) {
            const int at = atomicAdd(&whos, 1);
            who[at] = (uint16_t)j;
            atomicOr(&times[id], 1u);
          }
        }
    }
    for (int x = e0 + tid; x < e1; x += RT) {
      const uint32_t id = a.bias_id[x] - (uint32_t)id0;
      if (id < (uint32_t)span) atomicMax(&entry[id], x);
    }
    __syncthreads();
    listed = whos;
    __syncthreads();  // (the rows' values take its place)
    if (listed) {
      for (int i = i0 + wave; i < i1; i += RT / 64)
        for (int x = 0; x < listed; x += 64) {
          const int j = who[min(x + lane, listed - 1)];
          const uint32_t word = a.mask[(size_t)b * a.mask_stride + (size_t)i * a.words + j / 32];
          const uint64_t seen = __ballot(x + lane < listed && (word >> (j % 32) & 1));
          if (lane == 0) paths[i - i0][x / 64] = seen;
        }
      __syncthreads();
      for (int x = tid; x < listed; x += RT) who[x] = (uint16_t)(a.tokens[(size_t)b * a.rows + who[x]] - (uint32_t)id0);
      __syncthreads();
      token = who[min(lane, listed - 1)];
      if (lane >= listed || token / V % RT / 64 != wave) token = -1;
    }
#pragma unroll
    for (int e = 0; e < PER; e++) {
      const int l = mine(e), at = entry[l];
      const uint64_t all = __ballot(times[l] || at >= 0);
      if (all >> lane & 1) list[WIDS * wave + changes + __popcll(all & ((1ull << lane) - 1ull))] = (uint16_t)l;
      changes += __popcll(all);
      bias[l] = at >= 0 ? a.bias[at] : 0.0f;
    }
    in_order();
    one = lane < changes ? list[WIDS * wave + lane] : first;
    onebias = bias[one];
  }

  auto row = [&](auto all, Row &now, int i) {
    float v[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) v[e] = (float)now.x[e / V][e % V];
    uint32_t ok[G];
#pragma unroll
    for (int t = 0; t < G; t++) ok[t] = now.ok[t];
    load(all, now, min(i + 2, i1 - 1));
    if (changes) {
      // The tokens on node i's path among this wavefront's ids: one more of each (or one less).
      auto add = [&](uint32_t more) {
        if (token >= 0 && (paths[i - i0][0] >> lane & 1)) atomicAdd(&times[token], more);
        for (int x = 64 + lane; x < listed; x += 64) {
          const int id = who[x];
          if (id / V % RT / 64 == wave && (paths[i - i0][x / 64] >> lane & 1)) atomicAdd(&times[id], more);
        }
      };
      add(2u);
#pragma unroll
      for (int t = 0; t < PER / 4; t++)
        *(floatx4 *)(values + mine(4 * t)) = floatx4{v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]};
      in_order();
      auto change = [&](int l, float add) {
        const uint32_t c = times[l] >> 1;
        float y = values[l];
        if (c) y = ((y > 0.0f ? y / r : y * r) - f * (float)c) - p;
        values[l] = y + add;
      };
      if (lane < changes) change(one, onebias);
      for (int x = 64 + lane; x < changes; x += 64) {
        const int l = list[WIDS * wave + x];
        change(l, bias[l]);
      }
      in_order();
#pragma unroll
      for (int t = 0; t < PER / 4; t++) {
        const floatx4 y = *(const floatx4 *)(values + mine(4 * t));
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * t + e] = y[e];
      }
      add(0u - 2u);
      in_order();
    }
    if constexpr (ALLOW)
#pragma unroll
      for (int e = 0; e < PER; e++) {
        const uint32_t keep = (uint32_t)((int32_t)(ok[e / V] << (31 - e % V)) >> 31);
        v[e] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v[e]) & keep) | (0xff800000u & ~keep));
      }
    if constexpr (OUT) {
      T *out = (T *)a.out + (row0 + i) * a.ld + id0;
#pragma unroll
      for (int t = 0; t < G; t++) {
        const int l = first + V * RT * t, left = a.vocab - id0 - l;
        P w;
#pragma unroll
        for (int e = 0; e < V; e++) w[e] = (T)v[V * t + e];
        if constexpr (all) {
          __builtin_nontemporal_store(w, (typename Piece<T>::any *)(out + l));  // (not read again here)
        } else {
#pragma unroll
          for (int e = 0; e < V; e++)
            if (e < left) out[l + e] = w[e];
        }
      }
    }
    if (!a.part) return;
    float tops[G], best = -INFINITY;  // (ids that are not there hold −∞, as masked ones do)
#pragma unroll
    for (int t = 0; t < G; t++) {
      tops[t] = v[V * t];
#pragma unroll
      for (int e = 1; e < V; e++) tops[t] = fmaxf(tops[t], v[V * t + e]);
      best = fmaxf(best, tops[t]);
    }
    best = xlane::wave_max(best);
    // Its first place, which the others' mass against it leaves out.
    int at = INT_MAX;
    if (best > -INFINITY) {
#pragma unroll
      for (int t = G - 1; t >= 0; t--) {
        int e0 = V - 1;
#pragma unroll
        for (int e = V - 2; e >= 0; e--) e0 = v[V * t + e] == best ? e : e0;
        const uint64_t any = __ballot(tops[t] == best);
        const int l = any ? (int)__builtin_ctzll(any) : 0, place = V * (64 * wave + l + RT * t) + __builtin_amdgcn_readlane(e0, l);
        at = any ? place : at;
      }
#pragma unroll
      for (int e = 0; e < PER; e++) v[e] = at - first == V * RT * (e / V) + e % V ? -INFINITY : v[e];
    }
    float rest = 0.0f;
    const float m = best == -INFINITY ? 0.0f : best;
#pragma unroll
    for (int e = 0; e < PER; e++) rest += __expf(v[e] - m);
    rest = xlane::wave_sum(rest);
    if (lane == 0) {
      RulePart *p = a.part + ((row0 + i) * a.chunks + chunk) * (RT / 64) + wave;
      const RulePart x{best, rest, at == INT_MAX ? at : id0 + at, 0};
      if (a.done) store_part(p, x);
      else *p = x;
    }
  };
  auto rows = [&](auto all) {
    for (int i = i0;;) {
      row(all, even, i);
      if (++i == i1) return;
      row(all, odd, i);
      if (++i == i1) return;
    }
  };
  if (whole) rows(std::true_type{});
  else rows(std::false_type{});

  if (!a.done) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (this wavefront's parts are out)
  __syncthreads();
  int &last = *(int *)times, at = b * a.groups + i0 / a.group;
  if (tid == 0) last = atomicAdd(&a.done[at], 1) == a.chunks - 1;
  __syncthreads();
  if (!last) return;
  const int parts = a.chunks * (RT / 64);
  for (int i = i0 + wave; i < i1; i += RT / 64)
    join_row(a.part + (row0 + i) * parts, parts, lane, a.pick ? a.pick + row0 + i : nullptr, a.logprob ? a.logprob + row0 + i : nullptr);
  if (tid == 0) a.done[at] = 0;
}

__global__ __launch_bounds__(64) void rules_pick_kernel(const RulePart *part, const int32_t *counts, int rows, int parts,
                                                        uint32_t *pick, float *logprob) {
  const int row = blockIdx.x;
  if (counts && row % rows >= counts[row / rows]) return;
  join_row(part + (size_t)row * parts, parts, threadIdx.x, pick ? pick + row : nullptr, logprob ? logprob + row : nullptr);
}

template <typename T>
int rules_launch(wh_ctx *ctx, const RuleArgs &a, int grid) {
  if (a.allow && a.out) wh_launch(ctx, (rules_kernel<T, true, true>), grid, RT, 0, a);
  else if (a.allow) wh_launch(ctx, (rules_kernel<T, true, false>), grid, RT, 0, a);
  else if (a.out) wh_launch(ctx, (rules_kernel<T, false, true>), grid, RT, 0, a);
  else wh_launch(ctx, (rules_kernel<T, false, false>), grid, RT, 0, a);
  return wh_launched(ctx, "logit rules");
}

}  // namespace

int launch_logit_rules(wh_ctx *ctx, const wh_tree *t, const wh_rules *r, const void *logits, void *out, int vocab, size_t ld,
                       int f16, uint32_t *pick, float *logprob) {
  if (int rc = tree_check(ctx, "logit rules", t)) return rc;
  if (!r || !logits || (!out && !pick && !logprob) || vocab <= 0 || vocab > 1 << 28 || ld < (size_t)vocab)
    return wh_fail(ctx, WH_EARG, "logit rules: rules, logits, an output and rows of %d ids (%zu apart) are needed", vocab, ld);
  // (from without a history, too: penalties compare it with a text's length of zero)
  if ((r->history && (r->history_cols <= 0 || r->history_cols > 1 << 30)) || ((r->history || r->penalty) && r->from < 0))
    return wh_fail(ctx, WH_EARG, "logit rules: texts of %d ids from %d on", r->history_cols, r->from);
  if (r->bias_start && (!r->bias_id || !r->bias || r->bias_len < 0 || r->bias_len > 1 << 30))
    return wh_fail(ctx, WH_EARG, "logit rules: biases need their ids, values and number");
  if (r->penalty && t->mask && !t->tokens) return wh_fail(ctx, WH_EARG, "logit rules: the nodes' tokens are needed");
  if (((uintptr_t)r->penalty | (uintptr_t)r->history | (uintptr_t)r->bias_start | (uintptr_t)r->bias_id | (uintptr_t)r->bias |
       (uintptr_t)r->allow | (uintptr_t)pick | (uintptr_t)logprob) % 4 || ((uintptr_t)logits | (uintptr_t)out) % (f16 ? 2 : 4))
    return wh_fail(ctx, WH_EARG, "logit rules: misaligned arrays");
  const size_t nodes = (size_t)t->batch * t->rows;
  const int chunks = (vocab + IDS - 1) / IDS, parts = chunks * (RT / 64);
  // Rows per workgroup: about ten (fewer count the text too often, more leave the last workgroups alone: 61 rows of
  // 131071 f16 ids for 8 requests take 103, 92, 91, 95, 95 and 100 us with 4, 8, 10, 12, 16 and 32 of them; texts of 448 ids
  // and 24 rows would rather have 4: 31.2 us against 33.5), or so few that there are 5 workgroups a CU.
  const int cus = ctx->cus > 0 ? ctx->cus : 256;
  const size_t want = 5 * (size_t)cus, each = (size_t)chunks * t->batch;
  int groups = (int)std::min<size_t>(t->rows, std::max<size_t>((want + each - 1) / each, (t->rows + GROUP - 1) / GROUP));
  const int group = (t->rows + groups - 1) / groups;
  groups = (t->rows + group - 1) / group;
  if (each * groups >= (size_t)1 << 24) return wh_fail(ctx, WH_EARG, "logit rules: %zu rows of %d ids", nodes, vocab);
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "logit rules: %s", hipGetErrorString(e));
  RulePart *part = nullptr;
  if ((pick || logprob) && !(part = (RulePart *)wh_scratch(ctx, sizeof(RulePart) * parts * nodes))) return WH_EOOM;
  // Who joins the parts: up to a workgroup a CU their last one (a row of 51866 f32 ids 9.5 us, 12.7 with a second launch,
  // whose start costs more than the counting; 9 such rows 10.8 and 12.5); many more of them wait for each other's counts and
  // for their rows' stores before those (18 such rows 12.8 us counted, 12.5 in two launches, 48 of them 16.9 and 13.4; 10 to
  // 14, which two launches take as well, are still 11.1 to 12.3 counted, 12.6 in two).
  // Picks that lie in the tokens are written when all that read those are through: by a second launch, unless they take
  // the very places of tokens that one run of rows alone reads.
  const uintptr_t p0 = (uintptr_t)pick, t0 = (uintptr_t)t->tokens;
  const bool over = pick && t->tokens && p0 < t0 + 4 * nodes && t0 < p0 + 4 * nodes && (p0 != t0 || groups > 1);
  const RuleArgs a{t->n, t->count, t->tokens, t->mask, t->mask_stride, t->rows, (t->rows + 31) / 32, r->penalty, r->history,
                   r->history_cols, r->from, r->bias_start, r->bias_id, r->bias, r->bias_len, r->allow, logits, out, vocab,
                   chunks, group, groups, ld, part, pick, logprob,
                   part && !over && each * groups <= (size_t)cus && t->batch * groups <= ATTEND_HEADS ? ctx->attend_count : nullptr};
  {
    ProfScope prof(ctx, "logit_rules", 0.0, (double)nodes * vocab * (f16 ? 2 : 4) * (out ? 2 : 1));
    if (int rc = f16 ? rules_launch<_Float16>(ctx, a, (int)each * groups) : rules_launch<float>(ctx, a, (int)each * groups)) return rc;
  }
  if (!part || a.done) return WH_OK;
  ProfScope prof(ctx, "logit_pick", 0.0, (double)sizeof(RulePart) * parts * nodes);
  wh_launch(ctx, rules_pick_kernel, (int)nodes, 64, 0, (const RulePart *)part, t->count, t->rows, parts, pick, logprob);
  return wh_launched(ctx, "logit pick");
}
