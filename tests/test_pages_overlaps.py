"""Outputs that overlap what a call of sampled decoding over caches in pages reads, refused without a GPU as the calls of
test_pages_refusals are: by a C++ program with a context of its own, whose pointers are never followed."""

import os
import subprocess

import pytest

from test_pages_refusals import ROOT, SOURCE

CASES = {
    "norm": r'''
  norm("an output that reaches into the next row", "overlap", [&](Call &a) { a.stride = a.y_stride = 1024, a.y = at<void>(M + 4 * 513); });
  norm("an output of another stride", "overlap", [&](Call &a) { a.stride = 1024, a.y_stride = 1025, a.y = at<void>(M + 4 * 512); });
  norm("an output of the last row alone", "overlap", [&](Call &a) { a.y = at<void>(M + 4 * (79 * 512 + 511)); });
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
