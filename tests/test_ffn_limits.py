"""The sizes at which the feed-forward products stop, against what include/clblas_amd.h states: tests/cpp/ffn_limits_sanitize.cpp, built
for the CPU with AddressSanitizer and UBSan.  No GPU is needed."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc for the HIP host headers")
def test_largest_sizes_taken_and_smallest_refused(tmp_path):
    exe = str(tmp_path / "ffn_limits_sanitize")
    cmd = [HIPCC, "-std=c++17", "-O1", "-g", "-Wall", "-Wno-unused-function",
           "-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
           "-Xarch_host", "-fno-sanitize-recover=undefined", "--offload-arch=gfx950",
           os.path.join(ROOT, "clblas_amd", "csrc", "ffn_api.cpp"),
           os.path.join(ROOT, "tests", "cpp", "ffn_limits_sanitize.cpp"), "-o", exe]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip().endswith("ok"), out.stdout[-2000:] + out.stderr[-3000:]


def test_the_header_states_them():
    text = re.sub(r"\s*\*?\s+", " ", open(os.path.join(ROOT, "include", "clblas_amd.h")).read())
    for stated in ("N beyond 2^20 - 319 and K beyond 2^21 - 576", "Dimensions beyond 2^31 - 513 and leading dimensions beyond 2^31 are refused", "K beyond 131071"):
        assert stated in text, stated
