"""Outputs that overlap what a call of sampled decoding over caches in pages reads, refused without a GPU as the calls of
test_pages_refusals are: by a C++ program with a context of its own, whose pointers are never followed."""

import os
import subprocess

import pytest

from test_pages_refusals import ROOT, SOURCE

CASES = {
    "append": r'''
  auto apart = [](Call &a) { a.k = at<void>(8 * M), a.v = at<void>(16 * M); };
  append("queries into keys", "overlap", [&](Call &a) { apart(a), a.y = at<void>(8 * M); });
  append("queries into values", "overlap", [&](Call &a) { apart(a), a.y = at<void>(16 * M + 4 * 79 * 512 + 4 * 127); });
  append("queries behind themselves", "overlap", [&](Call &a) { apart(a), a.y = at<void>(M + 4); });
  append("queries before themselves", "overlap", [&](Call &a) { apart(a), a.y = at<void>(M - 4 * 255); });
  append("queries between the rows of keys, too long", "overlap", [&](Call &a) { apart(a), a.y = at<void>(8 * M + 4 * 257); });
  append("queries of another stride", "overlap", [&](Call &a) { apart(a), a.y = at<void>(8 * M + 4 * 128), a.y_stride = 520; });
  append("lengths into lengths", "n_out", [&](Call &a) { a.n_out = at<int32_t>(4100); });
  append("lengths before lengths", "n_out", [&](Call &a) { a.n_out = at<int32_t>(4092); });
  append("lengths into counts", "n_out", [&](Call &a) { a.t.count = at<int32_t>(8196); });
  append("lengths into what was kept", "n_out", [&](Call &a) { a.kept = at<int32_t>(8188); });
  append("lengths into paths", "n_out", [&](Call &a) { a.x = a.y = nullptr, a.path = at<int32_t>(8192 - 4 * 79); });
''',
    "read": r'''
  auto to = [](Call &a, size_t k, size_t v) { a.k = at<void>(k), a.v = at<void>(v); };
  read("keys and values in one place", "overlap", [&](Call &a) { to(a, M, M); });
  read("values in the last row of keys", "overlap", [&](Call &a) { to(a, M, M + 4 * (79 * 512 + 127)); });
  read("keys in the last row of values", "overlap", [&](Call &a) { to(a, M + 4 * (79 * 512 + 127), M); });
  read("values that reach into keys", "overlap", [&](Call &a) { to(a, M, M + 4 * (512 - 127)); });
  read("f16 values that reach into keys", "overlap", [&](Call &a) { to(a, M, M + 2 * 126), a.out16 = 1; });
''',
    "norm": r'''
  norm("an output that reaches into the next row", "overlap", [&](Call &a) { a.stride = a.y_stride = 1024, a.y = at<void>(M + 4 * 513); });
  norm("an output of another stride", "overlap", [&](Call &a) { a.stride = 1024, a.y_stride = 1025, a.y = at<void>(M + 4 * 512); });
  norm("an output of the last row alone", "overlap", [&](Call &a) { a.y = at<void>(M + 4 * (79 * 512 + 511)); });
''',
    "attend": r'''
  auto apart = [](Call &a) { a.k = at<void>(8 * M), a.v = at<void>(16 * M); };
  attend("outputs over queries", "overlap", [&](Call &a) { apart(a), a.o = at<void>(M); });
  attend("outputs over keys", "overlap", [&](Call &a) { apart(a), a.o = at<void>(8 * M); });
  attend("outputs over values", "overlap", [&](Call &a) { apart(a), a.o = at<void>(16 * M - 4 * (80 * 256 - 1)); });
  attend("f16 outputs over queries", "overlap", [&](Call &a) { apart(a), a.out16 = 1, a.o = at<void>(M - 2 * (80 * 256 - 2)); });
''',
    "probs": r'''
  probs("probabilities over logits", "overlap", [&](Call &a) { a.logits = a.probs = at<float>(M), a.probs_ld = 1001; });
  probs("probabilities of another stride", "overlap", [&](Call &a) { a.logits = at<float>(M), a.probs = at<float>(M + 4000), a.probs_ld = 1500; });
  probs("probabilities over f16 logits", "overlap", [&](Call &a) { a.in16 = 1, a.logits = at<void>(M), a.probs = at<float>(M - 4 * (79 * 1000 + 999)); });
''',
    "sample": r'''
  auto apart = [](Call &a) { a.probs = at<float>(M), a.drafts = at<float>(8 * M), a.u = at<float>(16 * M), a.picks = at<uint32_t>(32 * M), a.ld = 1000; };
  sample("picks over tokens", "overlap", [&](Call &a) { apart(a), a.t.tokens = a.picks; });
  sample("picks over random numbers", "overlap", [&](Call &a) { apart(a), a.picks = at<uint32_t>(16 * M + 4 * 79); });
  sample("picks over probabilities", "overlap", [&](Call &a) { apart(a), a.picks = at<uint32_t>(M + 4 * 79999); });
  sample("picks over drafts", "overlap", [&](Call &a) { apart(a), a.picks = at<uint32_t>(8 * M - 4 * 79); });
''',
}


@pytest.mark.parametrize("call", list(CASES))
def test_overlaps_are_refused(call, tmp_path):
    src, obj, exe = tmp_path / "main.cpp", tmp_path / "main.o", tmp_path / "main"
    src.write_text(SOURCE[:SOURCE.index("int main()")] + "int main() {\n" + CASES[call] + '  printf("%d calls, %d not refused\\n", calls, bad);\n  return bad != 0;\n}\n')
    hipcc = ["/opt/rocm/bin/hipcc", "--offload-arch=gfx950"]
    for args in (["-std=c++17", "-x", "hip", "--cuda-host-only", str(src), "-I", os.path.join(ROOT, "wavo_amd", "csrc"), "-c", "-o", str(obj)],
                 [str(obj), os.path.join(ROOT, "wavo_amd", "libwavo_hip.a"), "-o", str(exe)]):
        subprocess.run(hipcc + args, check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "calls, 0 not refused" in out.stdout
