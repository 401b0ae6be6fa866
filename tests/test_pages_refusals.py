"""The calls of sampled decoding over caches in pages that have to be refused, without a GPU: a C++ program with a context of its
own makes each bad call and checks its code and text.  Nothing is queued by a refused call, so the pointers stand for device
memory and are never followed.  And what the binding's structures keep alive."""

import gc
import os
import subprocess
import weakref

import pytest

import wavo_amd as wa
from test_tree_binding import buffer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r'''
#include <cstdio>
#include <cmath>
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
static const size_t M = (size_t)1 << 20;

struct Call {
  wh_tree t{2, 40, at<int32_t>(), nullptr, at<uint32_t>(), at<uint32_t>(), 80};
  wh_heads h{4, 2, 64, at<float>(), at<float>(), 1e-6f, at<float>(), 100, 64, 0};
  wh_pages p{at<void>(), 10, at<int32_t>(), 5, 5, 32, WH_Q4_0, 2, 64};
  const void *x = at<void>(M), *k = at<void>(M), *v = at<void>(M);
  void *y = at<void>(64 * M), *o = at<void>(64 * M);
  size_t stride = 512, y_stride = 512;
  int in16 = 0, out16 = 0, heads = 4;
  const int32_t *path = nullptr, *kept = nullptr;
  int32_t *n_out = at<int32_t>(8192);
  const void *logits = at<void>();
  float *probs = at<float>();
  const float *temperature = at<float>(), *drafts = at<float>(), *u = at<float>();
  uint32_t *picks = at<uint32_t>();
  int vocab = 1000;
  size_t ld = 1001, probs_ld = 1000;
  bool tree = true, given = true, paged = true;
  const wh_tree *T() { return tree ? &t : nullptr; }
  const wh_heads *H() { return given ? &h : nullptr; }
  const wh_pages *P() { return paged ? &p : nullptr; }
};
#define CALL(name, ...)                                                                  \
  template <typename F> static void name(const char *what, const char *text, F f) {     \
    Call a;                                                                              \
    f(a);                                                                                \
    refused(__VA_ARGS__, what, text);                                                    \
  }
CALL(norm, wh_head_norm(&ctx, a.T(), a.H(), a.x, a.stride, a.in16, a.y, a.y_stride, a.out16))
CALL(append, wh_page_append(&ctx, a.T(), a.H(), a.x, a.k, a.v, a.stride, a.in16, a.path, a.kept, a.P(), a.y, a.y_stride, a.out16, a.n_out))
CALL(read, wh_page_read(&ctx, a.T(), a.P(), (void *)a.k, (void *)a.v, a.stride, a.out16))
CALL(attend, wh_page_attend(&ctx, a.T(), a.x, a.k, a.v, a.stride, a.in16, a.P(), a.o, a.out16, a.heads))
CALL(probs, wh_logit_probs(&ctx, a.T(), a.logits, a.ld, a.in16, a.vocab, a.temperature, a.probs, a.probs_ld))
CALL(sample, wh_tree_sample(&ctx, a.T(), a.probs, a.drafts, a.vocab, a.ld, a.u, a.picks))
#define A [](Call &a)

int main() {
  norm("no tree", "tree", A { a.tree = false; });
  norm("no lengths", "tree", A { a.t.n = nullptr; });
  norm("rows past the most", "tree", A { a.t.rows = 1025, a.t.mask_stride = 0; });
  norm("no heads", "heads", A { a.given = false; });
  norm("heads of none", "heads", A { a.h.heads = 0; });
  norm("uneven heads", "heads", A { a.h.heads = 5; });
  norm("heads past the most", "heads", A { a.h.heads = a.h.kv_heads = 1025; });
  norm("heads of 60", "heads", A { a.h.hd = 60; });
  norm("heads of 264", "heads", A { a.h.hd = 264; });
  norm("eps below zero", "eps", A { a.h.eps = -1e-9f; });
  norm("eps that is none", "eps", A { a.h.eps = NAN; });
  norm("eps without end", "eps", A { a.h.eps = INFINITY; });
  norm("no positions", "rotation", A { a.h.positions = 0; });
  norm("a rotation of 12", "rotation", A { a.h.rot = 12; });
  norm("a rotation past the head", "rotation", A { a.h.rot = 72; });
  norm("a rotation of none", "rotation", A { a.h.rot = 0; });
  norm("misaligned gains", "aligned", A { a.h.q_gain = at<float>(4098); });
  norm("no rows", "needed", A { a.x = nullptr; });
  norm("no output", "needed", A { a.y = nullptr; });
  norm("rows too close", "apart", A { a.stride = 511; });
  norm("outputs too close", "apart", A { a.y_stride = 511; });
  norm("rows too far", "apart", A { a.stride = ((size_t)1 << 31) + 2; });
  norm("misaligned rows", "aligned", A { a.x = at<void>(M + 2); });
  norm("odd f16 rows", "aligned", A { a.in16 = 1, a.stride = 513; });
  norm("odd f16 outputs", "aligned", A { a.out16 = 1, a.y_stride = 513; });
  norm("in place of another type", "place", A { a.y = (void *)a.x, a.out16 = 1; });
  norm("in place of another stride", "place", A { a.y = (void *)a.x, a.y_stride = 514; });
  norm("an output in the rows", "overlaps", A { a.y = at<void>(M + 4); });
  norm("an output before the rows", "overlaps", A { a.y = at<void>(M - 4); });

  append("no tree", "tree", A { a.tree = false; });
  append("no heads", "heads", A { a.given = false; });
  append("no pages", "pages", A { a.paged = false; });
  append("pages of 8 bits", "supported", A { a.p.type = WH_Q8_0; });
  append("pages of 48", "supported", A { a.p.page = 48; });
  append("pages of 16", "supported", A { a.p.page = 16; });
  append("pages of 512", "supported", A { a.p.page = 512; });
  append("pages of heads of 40", "supported", A { a.p.hd = a.h.hd = a.h.rot = 40; });
  append("pages of heads of 160", "supported", A { a.p.hd = a.h.hd = 160, a.h.rot = 64; });
  append("pages of no heads", "supported", A { a.p.kv_heads = 0; });
  append("no pool", "pool", A { a.p.pool = nullptr; });
  append("no tables", "pool", A { a.p.table = nullptr; });
  append("no pages in the pool", "pool", A { a.p.pages = 0; });
  append("no columns", "pool", A { a.p.table_cols = 0; });
  append("positions past the most", "pool", A { a.p.table_cols = (1 << 19) + 1, a.p.table_stride = 0; });
  append("tables too close", "apart", A { a.p.table_stride = 4; });
  append("a misaligned pool", "aligned", A { a.p.pool = at<void>(4104); });
  append("misaligned tables", "aligned", A { a.p.table = at<int32_t>(4097); });
  append("pages of other heads", "into pages", A { a.p.kv_heads = 4; });
  append("pages of other sizes", "into pages", A { a.p.hd = 32; });
  append("no keys", "needed", A { a.k = nullptr; });
  append("no values", "needed", A { a.v = nullptr; });
  append("queries without their output", "needed", A { a.y = nullptr; });
  append("an output without queries", "needed", A { a.x = nullptr; });
  append("queries of a path", "needed", A { a.path = at<int32_t>(); });
  append("rows too close", "apart", A { a.stride = 255; });
  append("rows of keys too close", "apart", A { a.x = a.y = nullptr, a.stride = 127; });
  append("outputs too close", "apart", A { a.y_stride = 255; });
  append("misaligned keys", "aligned", A { a.k = at<void>(M + 2); });
  append("a misaligned path", "aligned", A { a.x = a.y = nullptr, a.path = at<int32_t>(4098); });
  append("odd f16 rows", "aligned", A { a.in16 = 1, a.stride = 513; });
  append("in place of another type", "place", A { a.y = (void *)a.x, a.in16 = 1; });
  append("lengths out in place", "n_out", A { a.n_out = (int32_t *)a.t.n; });
  append("lengths out over counts", "n_out", A { a.n_out = at<int32_t>(16384), a.t.count = a.n_out; });
  append("lengths out over what was kept", "n_out", A { a.kept = a.n_out; });
  append("rows past a launch", "one call", A { a.t.batch = 1 << 14, a.t.rows = 256, a.t.mask_stride = 0, a.h.heads = a.h.kv_heads = a.p.kv_heads = 1024, a.stride = 1024 * 64, a.y_stride = 1024 * 64; });

  read("no tree", "tree", A { a.tree = false; });
  read("no pages", "pages", A { a.paged = false; });
  read("no keys", "needed", A { a.k = nullptr; });
  read("no values", "needed", A { a.v = nullptr; });
  read("rows too close", "apart", A { a.stride = 127; });
  read("odd f16 rows", "aligned", A { a.out16 = 1, a.stride = 129; });
  read("rows past a launch", "one call", A { a.t.batch = 32768, a.t.rows = 128, a.t.mask_stride = 0, a.p.kv_heads = 410, a.stride = 410 * 64; });
  read("misaligned rows", "aligned", A { a.v = at<void>(M + 1); });

  attend("no tree", "tree", A { a.tree = false; });
  attend("masks too close", "masks", A { a.t.mask_stride = 79; });
  attend("no pages", "pages", A { a.paged = false; });
  attend("pages of 48", "supported", A { a.p.page = 48; });
  attend("no queries", "needed", A { a.x = nullptr; });
  attend("no output", "needed", A { a.o = nullptr; });
  attend("keys without values", "needed", A { a.v = nullptr; });
  attend("uneven heads", "heads", A { a.heads = 3; });
  attend("heads past the most", "heads", A { a.heads = 1026; });
  attend("rows too close", "apart", A { a.stride = 255; });
  attend("rows too far", "apart", A { a.stride = ((size_t)1 << 23) + 1; });
  attend("misaligned queries", "aligned", A { a.x = at<void>(M + 2); });
  attend("odd f16 rows", "aligned", A { a.in16 = 1, a.stride = 513; });
  attend("sequences past a launch", "one call", A { a.t.batch = 65536, a.t.rows = 1; });
  attend("heads past a launch", "one call", A { a.t.batch = 8192, a.t.rows = 64, a.t.mask_stride = 0, a.p.kv_heads = 64, a.heads = 64, a.stride = 4096; });

  probs("no tree", "tree", A { a.tree = false; });
  probs("no logits", "needed", A { a.logits = nullptr; });
  probs("no output", "needed", A { a.probs = nullptr; });
  probs("no ids", "needed", A { a.vocab = 0; });
  probs("ids past the most", "needed", A { a.vocab = (1 << 28) + 1, a.ld = a.probs_ld = 1 << 29; });
  probs("rows too close", "needed", A { a.ld = 999; });
  probs("outputs too close", "needed", A { a.probs_ld = 999; });
  probs("misaligned logits", "misaligned", A { a.logits = at<void>(4098); });
  probs("misaligned f16 logits", "misaligned", A { a.in16 = 1, a.logits = at<void>(4097); });
  probs("misaligned temperatures", "misaligned", A { a.temperature = at<float>(4098); });
  probs("rows past a launch", "one call", A { a.t.batch = 1 << 22, a.t.rows = 1; });

  sample("no tree", "tree", A { a.tree = false; });
  sample("no probabilities", "needed", A { a.probs = nullptr; });
  sample("no random numbers", "needed", A { a.u = nullptr; });
  sample("no picks", "needed", A { a.picks = nullptr; });
  sample("no tokens", "needed", A { a.t.tokens = nullptr; });
  sample("no ids", "needed", A { a.vocab = 0; });
  sample("rows too close", "needed", A { a.ld = 999; });
  sample("misaligned drafts", "misaligned", A { a.drafts = at<float>(4098); });
  sample("sequences past a launch", "one call", A { a.t.batch = 1 << 22, a.t.rows = 1; });
  sample("misaligned random numbers", "misaligned", A { a.u = at<float>(4097); });
  printf("%d calls, %d not refused\n", calls, bad);
  return bad != 0;
}
'''


def test_bad_calls_are_refused(tmp_path):
    src, obj, exe = tmp_path / "main.cpp", tmp_path / "main.o", tmp_path / "main"
    src.write_text(SOURCE)
    hipcc = ["/opt/rocm/bin/hipcc", "--offload-arch=gfx950"]
    for args in (["-std=c++17", "-x", "hip", "--cuda-host-only", str(src), "-I", os.path.join(ROOT, "wavo_amd", "csrc"), "-c", "-o", str(obj)],
                 [str(obj), os.path.join(ROOT, "wavo_amd", "libwavo_hip.a"), "-o", str(exe)]):
        subprocess.run(hipcc + args, check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "calls, 0 not refused" in out.stdout


@pytest.mark.parametrize("name", ["wh_head_norm", "wh_page_append", "wh_page_read", "wh_page_attend", "wh_logit_probs", "wh_tree_sample"])
def test_no_context(name):
    args = [0 if t in (wa._i, wa._sz) else None for t in wa.SIGNATURES[name][1]]
    assert getattr(wa.lib(), name)(*args) == wa.EARG


def test_page_bytes():
    assert wa.page_bytes(wa.Q4_0, 64, 8, 128) == 64 * 8 * 2 * 72  # 64 bytes of nibbles and 4 factors a head's key or value
    assert wa.page_bytes(wa.F16, 32, 3, 96) == 32 * 3 * 2 * 192
    assert [wa.page_bytes(*a) for a in ((wa.Q8_0, 64, 8, 128), (wa.F16, 33, 8, 128), (wa.F16, 0, 8, 128), (wa.F16, 64, 0, 128), (wa.F16, 64, 8, 100),
                                        (wa.F16, -64, 8, 128))] == [0] * 6


@pytest.mark.parametrize("make,names", [(lambda **kw: wa.Heads(2, 1, 64, **kw), ["q_gain", "k_gain", "table"]),
                                        (lambda **kw: wa.Pages(pages=3, table_cols=1, table_stride=1, page=32, type=wa.F16, kv_heads=1, hd=32, **kw),
                                         ["pool", "table"])], ids=["Heads", "Pages"])
def test_buffers_live_as_long_as_what_points_to_them(make, names):
    buffers = {x: buffer(4096 * (i + 1)) for i, x in enumerate(names)}
    alive = {x: weakref.ref(b) for x, b in buffers.items()}
    made = make(**buffers)
    del buffers
    gc.collect()
    assert [x for x in names if alive[x]() is None] == []
    assert [getattr(made, x) for x in names] == [4096 * (i + 1) for i in range(len(names))]
    del made
    gc.collect()
    assert [x for x in names if alive[x]() is not None] == []
