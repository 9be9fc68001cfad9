"""Calls of more threads than one launch holds (ha_mnb_fused, ha_mnb_logprobs), which go in parts of their rows: rows of each part
against 64 bits."""
import numpy as np
import pytest

import fused_ref as fr
import hybrid_attention as ha
import test_gpu_fused as tf
import test_gpu_logprobs as tl

pytestmark = pytest.mark.gpu


def some(M):
    return sorted({0, 1, M // 2 - 1, M // 2, M // 2 + 1, M - 17, M - 1})


@pytest.mark.parametrize("M", [98307, (1 << 17) + 5])  # (3.2 10^9 threads at once, and more than a launch holds)
def test_product(M):
    import torch
    N, K = 65536, 96  # (K is not of 64: the general kernel, 512 threads for 16 x 64 results)
    words, s, b, W = fr.weight(N, K, seed=30)
    rng = np.random.default_rng(31)
    a = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float16)).to(tf.DEV)
    w = tf.handle(words, s, b, N, K, (4, 32, False))
    out = torch.full((M + 1, N), 777.0, device=tf.DEV, dtype=torch.float16)
    w.fused(M, a, out, ha.Epilogue())
    torch.cuda.synchronize()
    assert (out[M] == 777.0).all()
    rows = some(M)
    want, off = fr.fused(a[rows].cpu().numpy(), W)
    tf.check(out[rows].cpu().numpy().astype(np.float64), want, off, K, ha.F16)


def test_log_probabilities():
    import torch
    M, V, K = 9001, 1 << 20, 96
    words, s, b, W = fr.weight(V, K, seed=32, std=2 / np.sqrt(K))
    rng = np.random.default_rng(33)
    a = rng.standard_normal((M, K)).astype(np.float16)
    targets = rng.integers(0, V, (M, 2)).astype(np.int32)
    got = tl.Call(tf.handle(words, s, b, V, K, (4, 32, False)), M, 0, 2, 5, 0.0, targets)(torch.from_numpy(a).to(tf.DEV))
    assert all(np.isfinite(x).all() for x in got.values())
    rows = some(M)
    tl.check({n: x[rows] for n, x in got.items()}, fr.logprobs(a[rows], W, 1.0, targets[rows], 5), 2, 5)


def test_stored_logits_in_parts():
    """More rows than have their logits in the workspace at a time."""
    import torch
    M, V, K, k = 8333, 32768, 64, 23
    words, s, b, W = fr.weight(V, K, seed=34, std=2 / np.sqrt(K))
    rng = np.random.default_rng(35)
    a = rng.standard_normal((M, K)).astype(np.float16)
    targets = rng.integers(0, V, (M, 2)).astype(np.int32)
    c = tl.Call(tf.handle(words, s, b, V, K, (4, 32, False)), M, 0, 2, k, 0.0, targets)
    assert c.ws.numel() == 1 << 30
    got = c(torch.from_numpy(a).to(tf.DEV))
    assert all(np.isfinite(x).all() for x in got.values())
    rows = sorted({*some(M), 8191, 8192, 8193})
    tl.check({n: x[rows] for n, x in got.items()}, fr.logprobs(a[rows], W, 1.0, targets[rows], k), 2, k)
