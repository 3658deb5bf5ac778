"""The argument checks of the feed-forward products, built for the CPU with AddressSanitizer and UBSan: hipcc compiles
clblas_amd/csrc/ffn_api.cpp for the host, the launchers behind it are stubs (tests/cpp/ffn_api_sanitize.cpp).  No GPU is needed."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc for the HIP host headers")
def test_checks_under_asan_ubsan(tmp_path):
    exe = str(tmp_path / "ffn_api_sanitize")
    cmd = [HIPCC, "-std=c++17", "-O1", "-g", "-Wall", "-Wno-unused-function",
           "-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
           "-Xarch_host", "-fno-sanitize-recover=undefined", "--offload-arch=gfx950",
           os.path.join(ROOT, "clblas_amd", "csrc", "ffn_api.cpp"),
           os.path.join(ROOT, "tests", "cpp", "ffn_api_sanitize.cpp"), "-o", exe]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip().endswith("ok"), out.stdout[-2000:] + out.stderr[-3000:]
