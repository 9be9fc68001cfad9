"""Log probabilities over a vocabulary (ha_mnb_logprobs) against 64 bits: formats, one row to many, vocabularies from one token
on, equal logits, near certain rows, targets that are no tokens, rows that are not finite, streams and captured graphs."""
import numpy as np
import pytest

import fused_ref as fr
import hybrid_attention as ha
from test_gpu_fused import FORMATS, dev, handle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Call:
    def __init__(self, w, M, n_vocab, T=0, k=0, scale=0.0, targets=None):
        import torch
        i32 = dict(device=DEV, dtype=torch.int32)
        self.M, self.w = M, w
        self.logp, self.top = torch.full((M, T), 7.0, device=DEV), torch.full((M, k), 7.0, device=DEV)
        self.entropy, self.lse = torch.full((M,), 7.0, device=DEV), torch.full((M,), 7.0, device=DEV)
        self.ids = torch.full((M, k), 7, **i32)
        self.p = ha.LogProbs(n_vocab=n_vocab, scale=scale, targets=dev(targets), n_targets=T, top_k=k, logp=self.logp if T else None,
                             entropy=self.entropy, lse=self.lse, top_ids=self.ids if k else None, top_logp=self.top if k else None)
        self.ws = torch.full((w.logprobs_bytes(M, self.p),), 255, device=DEV, dtype=torch.uint8)

    def __call__(self, a, stream=None):
        import torch
        self.w.logprobs(self.M, a, self.p, self.ws, stream=stream)
        torch.cuda.synchronize()
        return {n: getattr(self, n).cpu().numpy() for n in ("logp", "entropy", "lse", "ids", "top")}


def close(got, want, off):
    """f32 results: rounded once (2^-24 of them; 2^-23 allows the sum before it)."""
    err = np.abs(got.astype(np.float64) - want) - off - 2.0 ** -23 * np.abs(want) - 1e-12
    assert np.isfinite(got).all() and err.max() <= 0, "%.3g beyond the bound" % err.max()


def check(got, want, T, k):
    off = want["off"]
    if T:
        ok = np.isfinite(want["logp"])
        assert (np.isnan(got["logp"]) == ~ok).all()
        close(got["logp"][ok], want["logp"][ok], np.broadcast_to(off[:, None], ok.shape)[ok])
    close(got["lse"], want["lse"], off)
    close(got["entropy"], want["entropy"], want["entropy_off"])
    if k:
        assert (got["ids"] == want["ids"]).all()
        close(got["top"], want["top"], off[:, None])


def run(M, V, K, fmt=(4, 32, False), n_vocab=0, T=2, k=5, scale=1.0, lean=3.0, seed=0, std=None):
    words, s, b, W = fr.weight(V, K, *fmt, seed=seed, std=std or 2 / np.sqrt(K))
    rng = np.random.default_rng([seed, M, V, K])
    n = n_vocab or V
    t = rng.integers(0, n, M)
    a = (rng.standard_normal((M, K)) + lean * rng.random((M, 1)) * W[t] / (W[t] ** 2).sum(1, keepdims=True) * 4).astype(np.float16)
    targets = rng.integers(0, n, (M, T)).astype(np.int32)
    if T:
        targets[::2, 0] = t[::2]
    w = handle(words, s, b, V, K, fmt)
    got = Call(w, M, n_vocab, T, k, 0.0 if scale == 1.0 else scale, targets)(dev(a))
    check(got, fr.logprobs(a, W[:n], np.float32(scale).astype(np.float64), targets, k), T, k)
    w.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,V,K", [(1, 1000, 256), (7, 640, 512), (40, 1999, 128), (300, 1300, 256)])
def test_formats(fmt, M, V, K):
    run(M, V, K, fmt)


@pytest.mark.parametrize("M", [1, 2, 3, 15, 16, 17, 32, 33, 64, 65, 100, 128, 130, 257, 600])
def test_rows(M):
    run(M, 2100, 256, T=1, k=8)


@pytest.mark.parametrize("V", [1, 2, 5, 63, 64, 65, 127, 128, 129, 256, 257, 1023, 5000])
@pytest.mark.parametrize("M", [1, 20, 200])
def test_vocabularies(M, V):
    run(M, V, 128, k=min(V, 6))


@pytest.mark.parametrize("K", [32, 64, 96, 192, 576, 2048, 2080, 4096])
@pytest.mark.parametrize("M", [1, 30, 200])
def test_depths(M, K):
    run(M, 700, K)


@pytest.mark.parametrize("k", [0, 1, 2, 20, 32, 64])
@pytest.mark.parametrize("M", [1, 9, 150])
def test_top(M, k):
    run(M, 3000, 256, T=3, k=k)
    run(M, 64, 256, T=0, k=k)


@pytest.mark.parametrize("n_vocab", [1, 60, 64, 65, 900, 999])
@pytest.mark.parametrize("M", [1, 50, 200])
def test_padding_is_no_token(M, n_vocab):
    run(M, 1000, 256, n_vocab=n_vocab, k=min(5, n_vocab))


@pytest.mark.parametrize("scale", [0.25, 1.7, 8.0])
@pytest.mark.parametrize("M", [1, 40, 200])
def test_temperature(M, scale):
    run(M, 1500, 256, scale=scale)


@pytest.mark.parametrize("M", [1, 30, 200])
def test_near_certain(M):
    """Log probabilities near zero keep their digits."""
    run(M, 2000, 512, lean=9.0, T=1, k=3)
    run(M, 2000, 512, lean=30.0, T=1, k=3, seed=1)


def test_large_vocabulary():
    run(2, 151936, 256, T=4, k=20, n_vocab=151669)
    run(17, 40000, 512, (3, 64, True), T=1, k=40)
    run(140, 40000, 128, T=1, k=5)


@pytest.mark.parametrize("M", [1, 18, 140])
def test_equal_logits_come_by_number(M):
    """Rows of zeros (every logit 0), and rows of the table that are copies of one another."""
    V, K, k = 4000, 128, 40
    words, s, b, W = fr.weight(40, K, seed=4, std=0.2)
    pick = np.random.default_rng(1).integers(0, 40, V)
    a = np.random.default_rng(2).standard_normal((M, K)).astype(np.float16)
    a[::3] = 0
    w = handle(words[pick], s[pick], None, V, K, (4, 32, False))
    targets = np.zeros((M, 1), np.int32)
    got = Call(w, M, 0, 1, k, 0.0, targets)(dev(a))
    z = (a.astype(np.float64) @ W.T)[:, pick]
    want = np.argsort(-z, axis=1, kind="stable")[:, :k]
    assert (got["ids"] == want).all()
    lse = np.log(np.exp(z).sum(1))
    assert np.abs(got["entropy"][::3] - np.log(V)).max() < 2.0 ** -20 * np.log(V)
    assert np.abs(got["top"] - (np.take_along_axis(z, want, 1) - lse[:, None])).max() < 1e-5


@pytest.mark.parametrize("M", [1, 18, 140])
def test_neighbouring_alternatives(M):
    """The largest tokens side by side in one block, and in two."""
    V, K = 3000, 256
    words, s, b, W = fr.weight(V, K, seed=6)
    s[500:530] *= 4
    s[1000:1003] *= 5
    W = fr.mo.dequant(words, s, V, K)
    a = np.random.default_rng(7).standard_normal((M, K)).astype(np.float16)
    w = handle(words, s, None, V, K, (4, 32, False))
    check(Call(w, M, 0, 0, 30)(dev(a)), fr.logprobs(a, W, k=30), 0, 30)


@pytest.mark.parametrize("M", [1, 18, 140])
def test_targets_that_are_no_tokens(M):
    V, K = 300, 128
    words, s, b, W = fr.weight(V, K, seed=9)
    a = np.random.default_rng(3).standard_normal((M, K)).astype(np.float16)
    targets = np.tile(np.array([0, -1, 279, 280, 299, 300, 2 ** 31 - 1, -2 ** 31], np.int32), (M, 1))
    w = handle(words, s, None, V, K, (4, 32, False))
    check(Call(w, M, 280, 8, 2, 0.0, targets)(dev(a)), fr.logprobs(a, W[:280], 1.0, targets, 2), 8, 2)


@pytest.mark.parametrize("M", [2, 18, 140])
def test_rows_that_are_not_finite(M):
    """They are NaN throughout and leave the others alone; so is every row where a scale of the table is not finite."""
    V, K = 1000, 256
    words, s, b, W = fr.weight(V, K, seed=10)
    a = np.random.default_rng(4).standard_normal((M, K)).astype(np.float16)
    targets = np.full((M, 1), 3, np.int32)
    want = fr.logprobs(a, W, 1.0, targets, 4)
    bad = a.copy()
    bad[1, 5] = np.nan
    if M > 2:
        bad[7, 255] = -np.inf
    w = handle(words, s, None, V, K, (4, 32, False))
    c = Call(w, M, 0, 1, 4, 0.0, targets)
    got = c(dev(bad))
    lost = [1] + ([7] if M > 2 else [])
    fine = [m for m in range(M) if m not in lost]
    for n in ("logp", "entropy", "lse", "top"):
        assert np.isnan(got[n][lost]).all()
    assert (got["ids"][lost] == -1).all()
    check({n: v[fine] for n, v in got.items()}, {n: v[fine] for n, v in want.items()}, 1, 4)
    s2 = s.copy()
    s2[999, 3] = np.inf
    got = Call(handle(words, s2, None, V, K, (4, 32, False)), M, 0, 1, 4, 0.0, targets)(dev(a))
    assert np.isnan(got["entropy"]).all() and (got["ids"] == -1).all()
    got = Call(handle(words, s2, None, V, K, (4, 32, False)), M, 999, 1, 4, 0.0, targets)(dev(a))  # (that row is padding)
    assert np.isfinite(got["entropy"]).all()


def test_long_context_of_large_values():
    """Logits far from zero: only differences count."""
    V, K, M = 500, 1024, 20
    words, s, b, W = fr.weight(V, K, seed=12, std=1.0)
    a = (30 * np.random.default_rng(5).standard_normal((M, K))).astype(np.float16)
    w = handle(words, s, None, V, K, (4, 32, False))
    targets = np.arange(M, dtype=np.int32)[:, None]
    check(Call(w, M, 0, 1, 5, 0.0, targets)(dev(a)), fr.logprobs(a, W, 1.0, targets, 5), 1, 5)


@pytest.mark.parametrize("M", [1, 20, 200])
def test_same_bits_on_a_stream_and_in_a_graph(M):
    import torch
    V, K = 5000, 256
    words, s, b, W = fr.weight(V, K, seed=13)
    w = handle(words, s, None, V, K, (4, 32, False))
    a = torch.randn(M, K, device=DEV).half()
    targets = np.arange(M, dtype=np.int32)[:, None]
    one, two = Call(w, M, 0, 1, 10, 0.0, targets), Call(w, M, 0, 1, 10, 0.0, targets)
    torch.cuda.synchronize()
    first = one(a)
    st = torch.cuda.Stream()
    again = two(a, st.cuda_stream)
    assert all(np.array_equal(first[n], again[n]) for n in first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.logprobs(M, a, two.p, two.ws, stream=torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        a.copy_(torch.randn(M, K, device=DEV).half())
        two.ids.zero_()
        two.ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        got = {n: getattr(two, n).cpu().numpy() for n in ("logp", "entropy", "lse", "ids", "top")}
        want = one(a)
        assert all(np.array_equal(got[n], want[n]) for n in got), k


def test_two_calls_at_once():
    """Two streams, one handle, a workspace each."""
    import torch
    V, K, M = 20000, 512, 40
    words, s, b, W = fr.weight(V, K, seed=14)
    w = handle(words, s, None, V, K, (4, 32, False))
    a = [torch.randn(M, K, device=DEV).half() for _ in range(2)]
    calls = [Call(w, M, 0, 0, 10) for _ in range(2)]
    torch.cuda.synchronize()
    want = [c(x) for c, x in zip(calls, a)]
    st = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for c in calls:
            c.ids.zero_()
        torch.cuda.synchronize()
        for c, x, t in zip(calls, a, st):
            w.logprobs(M, x, c.p, c.ws, stream=t.cuda_stream)
        torch.cuda.synchronize()
        for c, v in zip(calls, want):
            assert np.array_equal(c.ids.cpu().numpy(), v["ids"]) and np.array_equal(c.lse.cpu().numpy(), v["lse"])


def test_no_workspace_beyond_its_bytes():
    """What lies behind the workspace and the outputs is left as it was."""
    import torch
    V, K, M = 1111, 128, 33
    words, s, b, W = fr.weight(V, K, seed=15)
    w = handle(words, s, None, V, K, (4, 32, False))
    c = Call(w, M, 0, 0, 3)
    n = c.ws.numel()
    c.ws = torch.full((n + 4096,), 99, device=DEV, dtype=torch.uint8)
    a = dev(np.random.default_rng(1).standard_normal((M, K)).astype(np.float16))
    got = c(a)
    assert (c.ws[n:] == 99).all()
    check(got, fr.logprobs(a.cpu().numpy(), W, k=3), 0, 3)


@pytest.mark.parametrize("M,V,k", [(10, 32768, 20), (64, 32700, 0), (300, 6000, 20), (260, 20000, 20), (257, 4097, 64)])
def test_stored_logits(M, V, k):
    """Vocabularies whose logits are stored: more of them than a thread keeps in registers, and fewer."""
    run(M, V, 128, k=k)


@pytest.mark.parametrize("M,V", [(3, 60000), (3, 9000), (300, 60000), (300, 3000)])
def test_repeats_bit_for_bit(M, V):
    """Candidates come in any order; with many equal maxima that order must not show."""
    words, s, b, _ = fr.weight(V, 128, seed=9)
    words[:] = words[np.arange(V) % 150]  # each logit some hundred times
    s[:] = s[np.arange(V) % 150]
    rng = np.random.default_rng(2)
    a = dev(rng.standard_normal((M, 128)).astype(np.float16))
    w = handle(words, s, b, V, 128, (4, 32, False))
    call = Call(w, M, 0, 2, 30, targets=rng.integers(0, V, (M, 2)).astype(np.int32))
    first = call(a)
    for _ in range(5):
        again = call(a)
        assert all(first[n].tobytes() == again[n].tobytes() for n in first)
    w.close()
