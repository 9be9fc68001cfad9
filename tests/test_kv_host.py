"""Host code of the paged 4-bit K/V cache (csrc/kv_host.cpp) on the CPU, against a HIP runtime that runs nothing
(tests/host/kv_calls.cpp)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CXX = "/opt/rocm/llvm/bin/clang++"  # (_Float16)
CSRC = os.path.join(ROOT, "strands-decider-web_amd", "csrc")


@pytest.mark.skipif(not os.path.exists(CXX), reason="clang++ is missing")
def test_host(tmp_path):
    exe = str(tmp_path / "kv_calls")
    r = subprocess.run([CXX, "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"),
                        "-I" + CSRC, "-Wno-unused-result", os.path.join(CSRC, "kv_host.cpp"),
                        os.path.join(ROOT, "tests", "host", "kv_calls.cpp"), "-o", exe, "-lpthread"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
