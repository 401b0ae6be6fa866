"""The calls over drafted tokens that have to be refused (wh_tree_attend, wh_logit_rules, wh_tree_accept),
without a GPU: a C++ program with a context of its own makes each bad call and checks its code and text.
Nothing is queued by a refused call, so the pointers stand for device memory and are never followed."""

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r'''
#include <cstdio>
#include <cstring>
#include "internal.h"

static wh_ctx ctx;
static int bad = 0, calls = 0;
static void refused(int rc, const char *what, const char *text) {
  calls++;
  if (rc != WH_EARG || !strstr(wh_last_error(&ctx), text)) bad++, printf("%s: code %d, \"%s\"\n", what, rc, wh_last_error(&ctx));
  ctx.error.clear();
}
template <typename T> static T *at(size_t a = 4096) { return (T *)a; }

struct Attend {
  wh_tree t{2, 40, at<int32_t>(), nullptr, at<uint32_t>(), at<uint32_t>(), 80};
  const void *q = at<void>(), *k = at<void>(), *v = at<void>();
  size_t stride = 960;
  int in16 = 0;
  const uint32_t *kv = at<uint32_t>();
  size_t kv_stride = 5 * 320;
  int cols = 5;
  void *o = at<void>();
  int out16 = 0, heads = 5, kv_heads = 5, hd = 64;
};
template <typename F> static void attend(const char *what, const char *text, F f, bool tree = true) {
  Attend a;
  f(a);
  refused(wh_tree_attend(&ctx, tree ? &a.t : nullptr, a.q, a.k, a.v, a.stride, a.in16, a.kv, a.kv_stride, a.cols, a.o, a.out16, a.heads,
                         a.kv_heads, a.hd), what, text);
}
struct RulesCall {
  wh_tree t{2, 40, at<int32_t>(), nullptr, at<uint32_t>(), at<uint32_t>(), 80};
  wh_rules r{at<float>(), at<uint32_t>(), 100, 0, at<int32_t>(), at<uint32_t>(), at<float>(), 7, at<uint32_t>()};
  const void *logits = at<void>();
  void *out = at<void>();
  int vocab = 1000;
  size_t ld = 1001;
  int f16 = 0;
  uint32_t *pick = at<uint32_t>();
  float *logprob = at<float>();
};
template <typename F> static void rules(const char *what, const char *text, F f, bool given = true) {
  RulesCall a;
  f(a);
  refused(wh_logit_rules(&ctx, &a.t, given ? &a.r : nullptr, a.logits, a.out, a.vocab, a.ld, a.f16, a.pick, a.logprob), what, text);
}
struct Accept {
  wh_tree t{2, 40, at<int32_t>(), nullptr, at<uint32_t>(), at<uint32_t>(), 80};
  wh_kept w{at<void>(), at<void>(), 96, 96 * 80, 0, at<uint32_t>(), 5 * 32, 10 * 32, 3, 32};
  const uint32_t *picks = at<uint32_t>();
  int cols = 5;
  int32_t *path = at<int32_t>(), *kept = at<int32_t>();
  uint32_t *next = at<uint32_t>();
  int32_t *n_out = at<int32_t>();
  uint32_t *history = at<uint32_t>();
  int history_cols = 5;
};
template <typename F> static void accept(const char *what, const char *text, F f) {
  Accept a;
  f(a);
  refused(wh_tree_accept(&ctx, &a.t, a.picks, &a.w, a.cols, a.path, a.kept, a.next, a.n_out, a.history, a.history_cols), what, text);
}

int main() {
  attend("no tree", "tree", [](Attend &) {}, false);
  attend("no sequences", "tree", [](Attend &a) { a.t.batch = 0; });
  attend("no rows", "tree", [](Attend &a) { a.t.rows = 0; });
  attend("rows past the most", "tree", [](Attend &a) { a.t.rows = 1025; a.t.mask_stride = 0; });
  attend("nodes past the most", "tree", [](Attend &a) { a.t.batch = 1 << 20; });
  attend("no lengths", "tree", [](Attend &a) { a.t.n = nullptr; });
  attend("masks too close", "masks", [](Attend &a) { a.t.mask_stride = 79; });
  attend("misaligned lengths", "aligned", [](Attend &a) { a.t.n = at<int32_t>(4098); });
  attend("no q", "needed", [](Attend &a) { a.q = nullptr; });
  attend("no cache", "needed", [](Attend &a) { a.kv = nullptr; });
  attend("no output", "needed", [](Attend &a) { a.o = nullptr; });
  attend("k without v", "needed", [](Attend &a) { a.v = nullptr; });
  attend("v without k", "needed", [](Attend &a) { a.k = nullptr; });
  attend("no heads", "shape", [](Attend &a) { a.heads = 0; });
  attend("no key heads", "shape", [](Attend &a) { a.kv_heads = 0; });
  attend("uneven heads", "shape", [](Attend &a) { a.kv_heads = 2; });
  attend("heads past the most", "shape", [](Attend &a) { a.heads = a.kv_heads = 1025; a.stride = 1 << 20; });
  attend("head size 0", "shape", [](Attend &a) { a.hd = 0; });
  attend("head size 66", "shape", [](Attend &a) { a.hd = 66; });
  attend("head size 132", "shape", [](Attend &a) { a.hd = 132; });
  attend("no positions", "shape", [](Attend &a) { a.cols = 0; });
  attend("rows too close", "apart", [](Attend &a) { a.stride = 319; });
  attend("rows too far", "apart", [](Attend &a) { a.stride = ((size_t)1 << 31) + 2; });
  attend("caches too close", "apart", [](Attend &a) { a.kv_stride--; });
  attend("misaligned q", "aligned", [](Attend &a) { a.q = at<void>(4098); });
  attend("misaligned cache", "aligned", [](Attend &a) { a.kv = at<uint32_t>(4097); });
  attend("odd f16 rows", "aligned", [](Attend &a) { a.in16 = 1, a.stride = 961; });
  attend("sequences past a launch", "in one call", [](Attend &a) { a.t.batch = 65536, a.t.rows = 1; });
  attend("heads past a launch", "in one call", [](Attend &a) {
    a.t.batch = 4096, a.t.rows = 64, a.t.mask_stride = 0, a.heads = a.kv_heads = 128, a.hd = 4, a.kv_stride = 0;
  });
  attend("positions past the most", "shape", [](Attend &a) { a.cols = (1 << 24) + 1, a.kv_stride = 0; });
  attend("rows just too far", "apart", [](Attend &a) { a.stride = ((size_t)1 << 23) + 1; });
  rules("no rules", "needed", [](RulesCall &) {}, false);
  rules("no logits", "needed", [](RulesCall &a) { a.logits = nullptr; });
  rules("no output", "needed", [](RulesCall &a) { a.out = nullptr, a.pick = nullptr, a.logprob = nullptr; });
  rules("no ids", "needed", [](RulesCall &a) { a.vocab = 0; });
  rules("ids past the most", "needed", [](RulesCall &a) { a.vocab = (1 << 28) + 1, a.ld = 1 << 29; });
  rules("rows too close", "needed", [](RulesCall &a) { a.ld = 999; });
  rules("no texts' size", "texts", [](RulesCall &a) { a.r.history_cols = 0; });
  rules("texts past the most", "texts", [](RulesCall &a) { a.r.history_cols = (1 << 30) + 1; });
  rules("biases past the most", "biases", [](RulesCall &a) { a.r.bias_len = (1 << 30) + 1; });
  rules("texts from -1", "texts", [](RulesCall &a) { a.r.from = -1; });
  rules("biases without ids", "biases", [](RulesCall &a) { a.r.bias_id = nullptr; });
  rules("biases without values", "biases", [](RulesCall &a) { a.r.bias = nullptr; });
  rules("biases without a number", "biases", [](RulesCall &a) { a.r.bias_len = -1; });
  rules("no tokens", "tokens", [](RulesCall &a) { a.t.tokens = nullptr; });
  rules("misaligned logits", "misaligned", [](RulesCall &a) { a.logits = at<void>(4098); });
  rules("misaligned f16 logits", "misaligned", [](RulesCall &a) { a.f16 = 1, a.logits = at<void>(4097); });
  rules("misaligned picks", "misaligned", [](RulesCall &a) { a.pick = at<uint32_t>(4098); });
  rules("rows past a launch", "rows of", [](RulesCall &a) { a.t.batch = 1 << 18, a.t.rows = 1, a.vocab = 1 << 20, a.ld = 1 << 20; });
  rules("no lengths", "tree", [](RulesCall &a) { a.t.n = nullptr; });
  accept("no tokens", "needed", [](Accept &a) { a.t.tokens = nullptr; });
  accept("no masks", "needed", [](Accept &a) { a.t.mask = nullptr; });
  accept("no picks", "needed", [](Accept &a) { a.picks = nullptr; });
  accept("no path", "needed", [](Accept &a) { a.path = nullptr; });
  accept("no kept", "needed", [](Accept &a) { a.kept = nullptr; });
  accept("no next", "needed", [](Accept &a) { a.next = nullptr; });
  accept("no n_out", "needed", [](Accept &a) { a.n_out = nullptr; });
  accept("no positions", "needed", [](Accept &a) { a.cols = 0; });
  accept("no texts' size", "needed", [](Accept &a) { a.history_cols = 0; });
  accept("misaligned path", "aligned", [](Accept &a) { a.path = at<int32_t>(4098); });
  accept("no keys", "bad", [](Accept &a) { a.w.k = nullptr; });
  accept("no values", "bad", [](Accept &a) { a.w.v = nullptr; });
  accept("no caches", "bad", [](Accept &a) { a.w.kv = nullptr; });
  accept("no layers", "bad", [](Accept &a) { a.w.layers = 0; });
  accept("odd rows", "bad", [](Accept &a) { a.w.d = 33; });
  accept("rows too close", "apart", [](Accept &a) { a.w.stride = 31; });
  accept("layers too close", "apart", [](Accept &a) { a.w.layer_stride = 31; });
  accept("caches too close", "apart", [](Accept &a) { a.w.kv_stride = 159; });
  accept("layers' caches too close", "apart", [](Accept &a) { a.w.kv_layer_stride = 159; });
  accept("misaligned keys", "aligned", [](Accept &a) { a.w.k = at<void>(4098); });
  accept("rows past a launch", "in one call", [](Accept &a) {
    a.t.batch = 1 << 20, a.t.rows = 1, a.t.mask_stride = 0, a.w.d = 1 << 16, a.w.stride = 1 << 16, a.w.layers = 1, a.w.kv_stride = 5 << 16;
  });
  accept("odd f16 rows", "aligned", [](Accept &a) { a.w.in16 = 1, a.w.stride = 97; });
  printf("%d calls, %d not refused\n", calls, bad);
  return bad != 0;
}
'''


def test_bad_calls_are_refused(tmp_path):
    lib = os.path.join(ROOT, "wavo_amd", "libwavo_hip.a")
    assert os.path.exists(lib), "build the library first (__graft_entry__.build)"
    src, exe = tmp_path / "main.cpp", tmp_path / "main"
    src.write_text(SOURCE)
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-std=c++17", "-x", "hip", "--cuda-host-only", str(src), "-I",
                    os.path.join(ROOT, "wavo_amd", "csrc"), "-c", "-o", str(tmp_path / "main.o")], check=True, capture_output=True,
                   timeout=300)
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", str(tmp_path / "main.o"), lib, "-o", str(exe)], check=True,
                   capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "calls, 0 not refused" in out.stdout


@pytest.mark.parametrize("name", ["wh_tree_attend", "wh_logit_rules", "wh_tree_accept"])
def test_no_context(name):
    import wavo_amd as wa

    args = [0 if t in (wa._i, wa._sz) else None for t in wa.SIGNATURES[name][1]]
    assert getattr(wa.lib(), name)(*args) == wa.EARG


def run_calls(tmp_path, calls):
    """The same program with other calls: its output, an error if one of them is not refused."""
    head = SOURCE[:SOURCE.index("int main() {")]
    tail = '  printf("%d calls, %d not refused\\n", calls, bad);\n  return bad != 0;\n}\n'
    src, obj, exe = tmp_path / "main.cpp", tmp_path / "main.o", tmp_path / "main"
    src.write_text(head + "int main() {\n" + calls + tail)
    hipcc = ["/opt/rocm/bin/hipcc", "--offload-arch=gfx950"]
    for args in (["-std=c++17", "-x", "hip", "--cuda-host-only", str(src), "-I", os.path.join(ROOT, "wavo_amd", "csrc"), "-c", "-o", str(obj)],
                 [str(obj), os.path.join(ROOT, "wavo_amd", "libwavo_hip.a"), "-o", str(exe)]):
        subprocess.run(hipcc + args, check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    return out.stdout


def test_texts_from_below_zero_are_refused_without_texts_too(tmp_path):
    """Penalties alone count the tree's tokens; a start below zero would have had the kernel count a text that is not there."""
    out = run_calls(tmp_path, r'''
  for (int from : {-1, -1000, INT32_MIN})
    for (int cols : {0, 100})
      rules("no texts, from below zero", "texts", [&](RulesCall &a) { a.r.history = nullptr, a.r.history_cols = cols, a.r.from = from; });
  rules("texts from the lowest", "texts", [](RulesCall &a) { a.r.from = INT32_MIN; });
''')
    assert "7 calls, 0 not refused" in out
