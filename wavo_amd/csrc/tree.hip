// A decoder step over trees of drafted tokens (include/wavo_hip.h, wh_tree): attention of every node over
// its sequence's f16 cache and the nodes that it sees, and the path of the tree that is kept.
#include <algorithm>
#include <climits>

#include "internal.h"
#include "xlane.h"

namespace {

__device__ __forceinline__ float half_bits(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }
__device__ __forceinline__ float number(const float *p, size_t i) { return p[i]; }
__device__ __forceinline__ float number(const _Float16 *p, size_t i) { return (float)p[i]; }

struct AttendArgs {
  const void *q, *k, *v;
  size_t stride;
  const uint32_t *kv;
  size_t kv_stride;
  void *o;
  const int32_t *n, *count;
  const uint32_t *mask;
  size_t mask_stride;
  int rows, words, cols, heads, group, hd;
  float scale;
};

constexpr int KEYS = 256;

// One workgroup per query head of a node: blocks of 256 keys, one per thread, with the running maximum and
// sum of the softmax; then a thread per value.
template <typename T, typename OT>
__global__ __launch_bounds__(KEYS) void attend_kernel(AttendArgs a) {
  __shared__ float qs[128], p[KEYS], red[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int head = blockIdx.x % a.heads, row = blockIdx.x / a.heads, b = row / a.rows, i = row % a.rows;
  const int n = min(max(a.n[b], 0), a.cols), count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows;
  if (i >= count) return;
  const int half = a.heads / a.group * a.hd / 2, pairs = a.hd / 2, kh = head / a.group;
  const uint32_t *kc = a.kv + (size_t)b * a.kv_stride, *vc = kc + (size_t)half * a.cols;
  const T *q = (const T *)a.q + (size_t)row * a.stride + head * a.hd;
  const size_t node0 = (size_t)b * a.rows * a.stride + kh * a.hd;
  if (tid < a.hd) qs[tid] = number(q, tid);
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  const int total = n + (a.mask && a.k ? count : 0);
  bool any = false;
  for (int j0 = 0; j0 < total; j0 += KEYS) {
    const int j = j0 + tid, u = j - n;
    bool see = j < n;
    if (!see && j < total) see = a.mask[(size_t)b * a.mask_stride + (size_t)i * a.words + u / 32] >> (u % 32) & 1;
    float s = -INFINITY;
    __syncthreads();
    if (see) {
      s = 0.0f;
      if (j < n) {
        for (int c = 0; c < pairs; c++) {
          const uint32_t w = kc[((size_t)kh * pairs + c) * a.cols + j];
          s += qs[2 * c] * half_bits(w & 0xffffu) + qs[2 * c + 1] * half_bits(w >> 16);
        }
      } else {
        const T *k = (const T *)a.k + node0 + (size_t)u * a.stride;
        for (int c = 0; c < a.hd; c++) s += qs[c] * (float)(_Float16)number(k, c);
      }
      s *= a.scale;
    }
    float bm = xlane::wave_max(s);
    if (lane == 0) red[wave] = bm;
    any |= __syncthreads_or(see) != 0;
    bm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mn = fmaxf(m, bm), m0 = mn == -INFINITY ? 0.0f : mn, old = __expf(m - m0);
    const float e = see ? __expf(s - m0) : 0.0f;
    p[tid] = see ? e : -1.0f;  // −1: not seen
    const float bl = xlane::wave_sum(e);
    if (lane == 0) red[4 + wave] = bl;
    __syncthreads();
    l = l * old + (red[4] + red[5] + red[6] + red[7]);
    acc *= old;
    m = mn;
    if (tid < a.hd)
      for (int x = 0; x < min(KEYS, total - j0); x++) {
        const int y = j0 + x;
        if (p[x] < 0.0f) continue;
        float val;
        if (y < n) {
          const uint32_t w = vc[(size_t)y * half + kh * pairs + tid / 2];
          val = half_bits(tid & 1 ? w >> 16 : w & 0xffffu);
        } else {
          val = (float)(_Float16)number((const T *)a.v + node0 + (size_t)(y - n) * a.stride, tid);
        }
        acc += p[x] * val;
      }
  }
  if (tid < a.hd) ((OT *)a.o)[((size_t)row * a.heads + head) * a.hd + tid] = (OT)(any ? acc / l : 0.0f);
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

// One workgroup per sequence: every node's parent (the highest bit below its own) and whether its token is
// the parent's pick; of a parent's agreeing children the first; then the walk from the root.
__global__ __launch_bounds__(256) void accept_kernel(AcceptArgs a) {
  __shared__ int child[TREE_ROWS], path[TREE_ROWS], kept;
  const int tid = threadIdx.x, b = blockIdx.x;
  const int n = min(max(a.n[b], 0), a.cols), count = a.count ? min(max(a.count[b], 0), a.rows) : a.rows;
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
    kept = k;
    a.kept[b] = k;
    if (count) a.next[b] = k ? picks[path[k - 1]] : tokens[0];
    a.n_out[b] = n + k;
  }
  __syncthreads();
  for (int i = tid; i < a.rows; i += 256) a.path[(size_t)b * a.rows + i] = i < kept ? path[i] : -1;
  if (a.history)
    for (int i = tid; i < kept; i += 256) a.history[(size_t)b * a.history_cols + n + i] = tokens[path[i]];
}

struct KeepArgs {
  const int32_t *path, *kept, *n_out;
  const void *k, *v;
  size_t stride, layer_stride;
  uint32_t *kv;
  size_t kv_stride, kv_layer_stride;
  int rows, cols, d, parts;
};

// The kept nodes' K and V into the caches: a thread per pair of values, K's pairs and then V's.
template <typename T>
__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a) {
  const int part = blockIdx.x % a.parts, b = blockIdx.x / a.parts, layer = blockIdx.y;
  const int i = part * 256 + threadIdx.x, half = a.d / 2;
  if (i >= a.d) return;
  const int kept = a.kept[b], n = a.n_out[b] - kept, c = i < half ? i : i - half;
  const T *x = (const T *)(i < half ? a.k : a.v) + layer * a.layer_stride + (size_t)b * a.rows * a.stride + 2 * c;
  uint32_t *y = a.kv + layer * a.kv_layer_stride + b * a.kv_stride;
  for (int s = 0; s < kept; s++) {
    const T *p = x + (size_t)a.path[(size_t)b * a.rows + s] * a.stride;
    const uint32_t lo = __builtin_bit_cast(uint16_t, (_Float16)p[0]), hi = __builtin_bit_cast(uint16_t, (_Float16)p[1]);
    y[i < half ? (size_t)c * a.cols + n + s : (size_t)half * a.cols + (size_t)(n + s) * half + c] = lo | hi << 16;
  }
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
  if (heads <= 0 || heads > ATTEND_HEADS || kv_heads <= 0 || heads % kv_heads || hd <= 0 || hd > 128 || hd % 4 || cols <= 0)
    return wh_fail(ctx, WH_EARG, "tree attention: bad shape (heads %d, key heads %d, head_dim %d, cols %d)", heads, kv_heads, hd,
                   cols);
  if (stride < (size_t)heads * hd || stride > (size_t)1 << 31)
    return wh_fail(ctx, WH_EARG, "tree attention: rows of %d queries %zu apart", heads * hd, stride);
  if (kv_stride && kv_stride < (size_t)cols * kv_heads * hd)
    return wh_fail(ctx, WH_EARG, "tree attention: caches of %zu words %zu apart", (size_t)cols * kv_heads * hd, kv_stride);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)kv | (uintptr_t)o) % 4 || (in16 && stride % 2))
    return wh_fail(ctx, WH_EARG, "tree attention: buffers and rows must be 4-byte aligned");
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "tree attention: %s", hipGetErrorString(e));
  const AttendArgs a{q, k, v, stride, kv, kv_stride, o, t->n, t->count, t->mask, t->mask_stride, t->rows, (t->rows + 31) / 32,
                     cols, heads, heads / kv_heads, hd, 1.0f / sqrtf((float)hd)};
  if ((size_t)t->batch * t->rows * heads >= (size_t)1 << 24)  // (a launch's threads fit 32 bits)
    return wh_fail(ctx, WH_EARG, "tree attention: %d heads of %d nodes in one call", heads, t->batch * t->rows);
  const int grid = t->batch * t->rows * heads;
  ProfScope prof(ctx, "tree_attend", 4.0 * grid * cols * hd, 4.0 * t->batch * cols * kv_heads * hd);
  if (in16 && out16) wh_launch(ctx, (attend_kernel<_Float16, _Float16>), grid, KEYS, 0, a);
  else if (in16) wh_launch(ctx, (attend_kernel<_Float16, float>), grid, KEYS, 0, a);
  else if (out16) wh_launch(ctx, (attend_kernel<float, _Float16>), grid, KEYS, 0, a);
  else wh_launch(ctx, (attend_kernel<float, float>), grid, KEYS, 0, a);
  return wh_launched(ctx, "tree attention");
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
    if (((uintptr_t)w->k | (uintptr_t)w->v | (uintptr_t)w->kv) % 4 || (w->in16 && (w->stride % 2 || w->layer_stride % 2)))
      return wh_fail(ctx, WH_EARG, "tree accept: buffers and rows must be 4-byte aligned");
  }
  if (hipError_t e = hipSetDevice(ctx->device)) return wh_fail(ctx, WH_EGPU, "tree accept: %s", hipGetErrorString(e));
  const AcceptArgs a{t->n, t->count, t->tokens, t->mask, picks, t->mask_stride, t->rows, (t->rows + 31) / 32, cols,
                     path, kept, next, n_out, history, history_cols};
  {
    ProfScope prof(ctx, "tree_accept", 0.0, 16.0 * t->batch * t->rows);
    wh_launch(ctx, accept_kernel, t->batch, 256, 0, a);
    if (int rc = wh_launched(ctx, "tree accept")) return rc;
  }
  if (!w) return WH_OK;
  const int parts = (w->d + 255) / 256;
  const KeepArgs ka{path, kept, n_out, w->k, w->v, w->stride, w->layer_stride, w->kv, w->kv_stride, w->kv_layer_stride,
                    t->rows, cols, w->d, parts};
  const dim3 grid(t->batch * parts, w->layers);
  ProfScope prof(ctx, "tree_keep", 0.0, 0.0);
  if (w->in16) wh_launch(ctx, keep_kernel<_Float16>, grid, 256, 0, ka);
  else wh_launch(ctx, keep_kernel<float>, grid, 256, 0, ka);
  return wh_launched(ctx, "tree keep");
}
