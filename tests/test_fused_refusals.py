"""What the products whose results are not stored as they are refuse (ha_mnb_fused, ha_mnb_logprobs): the host code on the CPU
against a HIP runtime that runs nothing (tests/host/fused_calls.cpp), forged handles, and tensors that a call could not read."""
import ctypes
import os
import subprocess

import pytest

import hybrid_attention as ha
from test_kv_refusals import Fake

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CXX = "/opt/rocm/llvm/bin/clang++"  # (_Float16)
CSRC = os.path.join(ROOT, "strands-decider-web_amd", "csrc")


@pytest.mark.skipif(not os.path.exists(CXX), reason="clang++ is missing")
def test_host(tmp_path):
    exe = str(tmp_path / "fused_calls")
    r = subprocess.run([CXX, "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"),
                        "-I" + CSRC, "-Wno-unused-result", os.path.join(CSRC, "fused_host.cpp"),
                        os.path.join(ROOT, "tests", "host", "fused_calls.cpp"), "-o", exe, "-lpthread"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_handles():
    lib = ha.load_library()
    buf = (ctypes.c_uint32 * 64)()
    buf[0] = 0x48414D4E
    n = ctypes.c_size_t(7)
    for h in (None, ctypes.cast(buf, ctypes.c_void_p)):
        assert lib.ha_mnb_fused(h, 1, None, None, None, None) == ha.HA_ERR_HANDLE
        assert lib.ha_mnb_logprobs(h, 1, None, None, None, 0, None) == ha.HA_ERR_HANDLE
        assert lib.ha_mnb_logprobs_bytes(h, 1, None, ctypes.byref(n)) == ha.HA_ERR_HANDLE and n.value == 0
    assert buf[0] == 0x48414D4E


class Weight(ha.MnbWeight):
    """A weight without memory: its calls check their tensors and end at the library's look at the handle."""

    def __init__(self, N, K):
        ha.load_library()
        self.N, self.K, self._device, self._h = N, K, 0, None


@pytest.fixture
def no_torch(monkeypatch):
    import sys
    monkeypatch.setitem(sys.modules, "torch", None)  # (types are compared as texts)


def ends_at_the_handle(call):
    with pytest.raises(ha.HAError) as ei:
        call()
    assert ei.value.code == ha.HA_ERR_HANDLE


BAD = [dict(gpu=1), dict(cuda=False), dict(contiguous=False), dict(dtype="bfloat16")]


def test_product_tensors(no_torch):
    w = Weight(100, 64)
    a, out = Fake(3 * 64), Fake(300)
    ends_at_the_handle(lambda: w.fused(3, a, out, ha.Epilogue()))
    ends_at_the_handle(lambda: w.fused(3, 4096, 8192, ha.Epilogue(residual=4096, bias=4096)))
    for bad in BAD:
        with pytest.raises(TypeError):
            w.fused(3, Fake(3 * 64, **bad), out, ha.Epilogue())
    for bad in [dict(gpu=1), dict(cuda=False), dict(dtype="float32")]:
        with pytest.raises(TypeError):
            w.fused(3, a, Fake(300, **bad), ha.Epilogue())
    with pytest.raises(TypeError):
        w.fused(3, Fake(3 * 64 - 1), out, ha.Epilogue())
    with pytest.raises(TypeError):
        w.fused(3, a, Fake(299), ha.Epilogue())
    with pytest.raises(TypeError):
        w.fused(3, a, Fake(149), ha.Epilogue(gated=True))
    ends_at_the_handle(lambda: w.fused(3, a, Fake(150), ha.Epilogue(gated=True)))
    with pytest.raises(TypeError):
        w.fused(3, a, out, ha.Epilogue(bias=Fake(99, "float32")))
    with pytest.raises(TypeError):
        w.fused(3, a, out, ha.Epilogue(bias=Fake(100)))
    with pytest.raises(TypeError):
        w.fused(3, a, out, ha.Epilogue(residual=Fake(300)))  # (f32 unless said)
    ends_at_the_handle(lambda: w.fused(3, a, out, ha.Epilogue(residual=Fake(300), residual_dtype=ha.F16, bias=Fake(100, "float32"))))
    with pytest.raises(ValueError):
        ha.Epilogue(act="relu")
    e = ha.Epilogue(residual=Fake(300, "float32"))  # kept for more rows than its residual has
    ends_at_the_handle(lambda: w.fused(3, a, out, e))
    with pytest.raises(TypeError):
        w.fused(4, Fake(256), Fake(400), e)


def test_logprobs_tensors(no_torch):
    w = Weight(100, 64)
    a, ws = Fake(3 * 64), Fake(10000)
    ws.element_size = lambda: 1
    f, i = (lambda n: Fake(n, "float32")), (lambda n: Fake(n, "int32"))
    good = dict(targets=i(6), n_targets=2, logp=f(6), entropy=f(3), lse=f(3), top_k=4, top_ids=i(12), top_logp=f(12))
    ends_at_the_handle(lambda: w.logprobs(3, a, ha.LogProbs(**good), ws))
    for name, n, other in [("targets", 5, f), ("logp", 5, i), ("entropy", 2, i), ("lse", 2, i), ("top_ids", 11, f), ("top_logp", 11, i)]:
        for bad in (good[name].__class__(n, str(good[name].dtype)[6:]), other(n + 1)):
            with pytest.raises(TypeError):
                w.logprobs(3, a, ha.LogProbs(**{**good, name: bad}), ws)
    for bad in BAD:
        with pytest.raises(TypeError):
            w.logprobs(3, Fake(3 * 64, **bad), ha.LogProbs(**good), ws)
    with pytest.raises(TypeError):
        w.logprobs(3, a, ha.LogProbs(**good), Fake(10000, cuda=False))
    ends_at_the_handle(lambda: w.logprobs_bytes(3, ha.LogProbs(**good)))
