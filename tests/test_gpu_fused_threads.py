"""Log probabilities from several threads at once, with calls that need little and much LDS of the same kernels: each as if alone."""
import threading

import numpy as np
import pytest

import fused_ref as fr
import test_gpu_logprobs as tl

pytestmark = pytest.mark.gpu


def test_calls_of_many_sizes():
    import torch
    K, V = 2048, 40000
    words, s, b, _ = fr.weight(V, K, seed=50)
    w = tl.handle(words, s, b, V, K, (4, 32, False))
    rng = np.random.default_rng(51)
    calls = []
    for M, T, k in ((16, 1024, 64), (12, 0, 40), (13, 500, 64), (16, 1024, 1)):
        targets = rng.integers(0, V, (M, T)).astype(np.int32)
        calls.append((tl.Call(w, M, 0, T, k, 0.0, targets), tl.dev(rng.standard_normal((M, K)).astype(np.float16))))
    want = [c(a) for c, a in calls]
    wrong = []

    def run(i):
        c, a = calls[i]
        st = torch.cuda.Stream()
        try:
            for _ in range(20):
                w.logprobs(c.M, a, c.p, c.ws, stream=st.cuda_stream)
            st.synchronize()
        except Exception as e:  # noqa: BLE001 (a thread's failure is the test's)
            wrong.append((i, e))
    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong
    for (c, _), x in zip(calls, want):
        for n in x:
            assert np.array_equal(getattr(c, n).cpu().numpy(), x[n], equal_nan=True), n


def test_a_graph_of_a_call_with_much_lds():
    """Captured and replayed with the program's own calls between: 128 KiB of rows in LDS, 1024 targets and the 64 largest in the join."""
    import torch
    K, V, M = 4096, 40000, 16
    words, s, b, _ = fr.weight(V, K, seed=52)
    w = tl.handle(words, s, b, V, K, (4, 32, False))
    targets = np.random.default_rng(53).integers(0, V, (M, 1024)).astype(np.int32)
    a = torch.randn(M, K, device=tl.DEV).half()
    one, two = (tl.Call(w, M, 0, 1024, 64, 0.0, targets) for _ in range(2))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):  # (nothing ran before it)
        w.logprobs(M, a, two.p, two.ws, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        a.copy_(torch.randn(M, K, device=tl.DEV).half())
        g.replay()
        torch.cuda.synchronize()
        want = one(a)
        for n in want:
            assert np.array_equal(getattr(two, n).cpu().numpy(), want[n]), n
