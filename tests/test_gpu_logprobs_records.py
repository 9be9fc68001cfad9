"""Log probabilities over vocabularies whose logits are not stored (above 32768 tokens) against 64 bits: every kernel that makes records and
every form of the join, last blocks of 1 to 64 tokens, and what the records themselves have to carry: equal logits, several of the
largest in one block, near certain rows, padding, rows that are not finite. tests/test_fused_coverage.py checks that the sizes here
reach all kernels."""
import functools

import numpy as np
import pytest

import fused_ref as fr
from test_gpu_fused_kernels import FORMATS
from test_gpu_logprobs import DEV, Call, check, close, dev, handle

pytestmark = pytest.mark.gpu
V = 33000  # 515 blocks and 40 tokens
# rows and K: the kernel of up to 16 rows (whole 256 k), tiles of 32 to 128 rows x 128 or 256 tokens, the general kernel (96; 192 with groups of 64)
SIZES = [(1, 256), (2, 512), (3, 1024), (16, 256), (17, 256), (40, 128), (61, 1152), (90, 128), (128, 128), (250, 1152), (1, 96), (5, 96), (45, 96)]
# 512 and 256 threads a row over records; 512, 256 and 1024 over logits
JOINS = [(257, 140001, 64), (257, 33001, 64), (300, 5000, 64), (300, 4000, 64), (20, 4000, 64)]
SOME = [(1, 256), (9, 256), (18, 128), (61, 128), (140, 128), (250, 128), (3, 96), (40, 96)]


def deep(K, fmt):
    """K = 96 stands for a K that the fast kernels do not take; 64 for a small one."""
    return K if fmt[1] == 32 else {96: 192, 64: 128}.get(K, K)


def cases():
    """(rows, vocabulary, K, format) of test_formats and test_joins."""
    return ([(M, V, deep(K, fmt), fmt) for fmt in FORMATS for M, K in SIZES] + [(M, V_, deep(K, fmt), fmt) for fmt in FORMATS for M, V_, K in JOINS])


@functools.lru_cache(4)
def table(V, K, fmt, seed=0):
    words, s, b, W = fr.weight(V, K, *fmt, seed=seed, std=2 / np.sqrt(K))
    return words, s, b, W


def rows_of(M):
    """All rows, or a hundred of them, the first and last 33 among them."""
    if M <= 140:
        return np.arange(M)
    return np.unique(np.concatenate([np.arange(33), np.arange(M - 33, M), np.random.default_rng(M).integers(0, M, 40)]))


def compare(got, a, W, scale, targets, k):
    M = len(a)
    r = rows_of(M)
    want = fr.logprobs(a[r], W, np.float32(scale).astype(np.float64), None if targets is None else targets[r], k)
    for n in ("entropy", "lse"):
        assert np.isfinite(got[n]).all()
    check({n: x[r] for n, x in got.items()}, want, 0 if targets is None else targets.shape[1], k)


def leaning(M, K, W, n, lean, seed):
    """Rows that lean, each by as much as it likes, towards a token's row."""
    rng = np.random.default_rng([seed, M, K])
    t = rng.integers(0, n, M)
    a = (rng.standard_normal((M, K)) + lean * rng.random((M, 1)) * W[t] / (W[t] ** 2).sum(1, keepdims=True) * 4).astype(np.float16)
    return a, t


def run(M, K, fmt=(4, 32, False), V=V, n_vocab=0, T=2, k=5, scale=1.0, lean=3.0, seed=0):
    words, s, b, W = table(V, K, fmt)
    n = n_vocab or V
    a, t = leaning(M, K, W, n, lean, seed)
    targets = np.random.default_rng(seed).integers(0, n, (M, T)).astype(np.int32)
    if T:
        targets[::2, 0] = t[::2]
    w = handle(words, s, b, V, K, fmt)
    got = Call(w, M, n_vocab, T, k, 0.0 if scale == 1.0 else scale, targets)(dev(a))
    compare(got, a, W[:n], scale, targets, k)
    w.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K", SIZES)
def test_formats(M, K, fmt):
    run(M, deep(K, fmt), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,V,K", JOINS)
def test_joins(M, V, K, fmt):
    run(M, deep(K, fmt), fmt, V=V, k=7)


@pytest.mark.parametrize("n_vocab", [32769, 32770, 32800, 32831, 32832, 32833, 32895, 32896, 32897, 33023, 33024, 33100])
@pytest.mark.parametrize("M,K", [(1, 256), (20, 128), (61, 128), (140, 128), (250, 128), (5, 96)])
def test_last_blocks_and_padding(M, K, n_vocab):
    """Last blocks of 1 to 64 tokens, in tiles of 128 and 256 tokens; the table's rows behind them are no tokens."""
    run(M, K, V=33100, n_vocab=n_vocab if n_vocab < 33100 else 0, k=6)


@pytest.mark.parametrize("k", [0, 1, 2, 20, 40, 64])
@pytest.mark.parametrize("M,K", [(1, 256), (9, 256), (61, 128), (140, 128), (250, 128)])
def test_top(M, K, k):
    run(M, K, T=3 if k else 0, k=k, seed=k)


@pytest.mark.parametrize("scale", [0.25, 1.7, 8.0])
@pytest.mark.parametrize("M,K", SOME)
def test_temperature(M, K, scale):
    run(M, K, scale=scale, seed=3)


@pytest.mark.parametrize("M,K", SOME)
def test_near_certain(M, K):
    run(M, K, lean=9.0, T=1, k=3, seed=1)
    run(M, K, lean=30.0, T=1, k=3, seed=2)


@pytest.mark.parametrize("M,K", SOME)
def test_equal_logits_come_by_number(M, K):
    """Rows of zeros (every logit 0), and rows of the table that are copies of one another, in a block and in many."""
    k = 40
    words, s, b, W = fr.weight(40, K, seed=4, std=0.2)
    pick = np.random.default_rng(1).integers(0, 40, V)
    pick[6400:6464] = pick[6400]  # a block of one row, and the last
    pick[32960:] = pick[6400]
    a = np.random.default_rng(2).standard_normal((M, K)).astype(np.float16)
    a[::3] = 0
    w = handle(words[pick], s[pick], None, V, K, (4, 32, False))
    got = Call(w, M, 0, 1, k, 0.0, np.zeros((M, 1), np.int32))(dev(a))
    z = (a.astype(np.float64) @ W.T)[:, pick]
    want = np.argsort(-z, axis=1, kind="stable")[:, :k]
    assert (got["ids"] == want).all()
    lse = np.log(np.exp(z).sum(1))
    off = fr.logprobs(a, W[pick])["off"]
    close(got["lse"], lse, off)
    assert np.abs(got["entropy"][::3] - np.log(V)).max() < 2.0 ** -20 * np.log(V)
    close(got["top"], np.take_along_axis(z, want, 1) - lse[:, None], off[:, None])


@pytest.mark.parametrize("fmt", [(4, 32, False), (4, 32, True), (3, 32, False), (2, 32, True)])
@pytest.mark.parametrize("M,K", SOME)
def test_several_of_the_largest_in_a_block(M, K, fmt):
    """Two, three, and thirty tokens of a block among the largest, two at its ends, and some of the last block, which is cut."""
    words, s, b, _ = fr.weight(V, K, *fmt, seed=6)
    more = np.concatenate([[640 + 3, 640 + 50], 6400 + np.array([0, 31, 63]), 12800 + np.arange(20, 50), [V - 1, V - 2, V - 40]])
    s[more] *= 4
    if b is not None:
        b[more] *= 4
    W = fr.mo.dequant(words, s, V, K, *fmt, b)
    a = np.random.default_rng(7).standard_normal((M, K)).astype(np.float16)
    w = handle(words, s, b, V, K, fmt)
    for k in (2, 30):
        compare(Call(w, M, 0, 0, k)(dev(a)), a, W, 1.0, None, k)


@pytest.mark.parametrize("M,K", SOME)
def test_targets_that_are_no_tokens(M, K):
    words, s, b, W = table(V, K, (4, 32, False))
    a = np.random.default_rng(3).standard_normal((M, K)).astype(np.float16)
    targets = np.tile(np.array([0, -1, V - 21, V - 20, V - 1, V, 2 ** 31 - 1, -2 ** 31], np.int32), (M, 1))
    w = handle(words, s, None, V, K, (4, 32, False))
    got = Call(w, M, V - 20, 8, 2, 0.0, targets)(dev(a))
    compare(got, a, W[:V - 20], 1.0, targets, 2)
    # logp in the targets' own place, as a call that asks for the same without (top_k says how many columns' values come from 64 bits)
    import torch
    import hybrid_attention as ha
    want, t = Call(w, M, V - 20, 8, 0, 0.0, targets)(dev(a))["logp"], dev(targets)
    p = ha.LogProbs(n_vocab=V - 20, targets=t, n_targets=8, logp=t.view(torch.float32))
    w.logprobs(M, dev(a), p, torch.empty(w.logprobs_bytes(M, p), device=DEV, dtype=torch.uint8))
    torch.cuda.synchronize()
    assert np.array_equal(t.view(torch.float32).cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("M,K", SOME)
def test_rows_that_are_not_finite(M, K, bad):
    """They are NaN throughout and leave the others alone; so is every row where a scale of the table is not finite: in a block's first
    column, in one in its middle, in the last token."""
    words, s, b, W = table(V, K, (4, 32, False))
    a = np.random.default_rng(4).standard_normal((M, K)).astype(np.float16)
    lost = sorted({M // 2, M - 1})
    x = a.copy()
    x[lost, 5] = bad
    w = handle(words, s, None, V, K, (4, 32, False))
    got = Call(w, M, 0, 1, 4, 0.0, np.full((M, 1), 3, np.int32))(dev(x))
    for n in ("logp", "entropy", "lse", "top"):
        assert np.isnan(got[n][lost]).all()
    assert (got["ids"][lost] == -1).all()
    fine = [m for m in range(M) if m not in lost][:60]
    if fine:
        check({n: v[fine] for n, v in got.items()}, fr.logprobs(a[fine], W, 1.0, np.full((len(fine), 1), 3), 4), 1, 4)
    for at in (6400, 6433, V - 1):
        s2 = s.copy()
        s2[at, K // 64] = bad
        w = handle(words, s2, None, V, K, (4, 32, False))
        got = Call(w, M, 0, 1, 4, 0.0, np.full((M, 1), 3, np.int32))(dev(a))
        assert np.isnan(got["entropy"]).all() and np.isnan(got["lse"]).all() and (got["ids"] == -1).all()
    got = Call(w, M, V - 1, 1, 4, 0.0, np.full((M, 1), 3, np.int32))(dev(a))  # (that row is padding)
    assert np.isfinite(got["entropy"]).all()


@pytest.mark.parametrize("M,K", SOME)
def test_large_values(M, K):
    """Logits far from zero: only differences count."""
    words, s, b, W = table(V, K, (4, 32, False))
    a = (300 * np.random.default_rng(5).standard_normal((M, K))).astype(np.float16)
    targets = np.arange(M, dtype=np.int32)[:, None]
    compare(Call(handle(words, s, None, V, K, (4, 32, False)), M, 0, 1, 5, 0.0, targets)(dev(a)), a, W, 1.0, targets, 5)


@pytest.mark.parametrize("M,K", SOME)
def test_same_bits_on_a_stream_and_in_a_graph(M, K):
    import torch
    words, s, b, W = table(V, K, (4, 32, False))
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


@pytest.mark.parametrize("M,K", SOME)
def test_nothing_behind_the_workspace_and_the_outputs(M, K):
    import torch
    words, s, b, W = table(V, K, (4, 32, False))
    w = handle(words, s, None, V, K, (4, 32, False))
    c = Call(w, M, 0, 0, 3)
    n = -(-V // 64) * 16 * M
    assert c.ws.numel() >= n
    c.ws = torch.full((n + 4096,), 99, device=DEV, dtype=torch.uint8)
    a = np.random.default_rng(1).standard_normal((M, K)).astype(np.float16)
    got = c(dev(a))
    assert (c.ws[n:] == 99).all()
    compare(got, a, W, 1.0, None, 3)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K", [(2, 256), (40, 128), (5, 96)])
def test_subnormal_operands(M, K, fmt):
    """Rows and scales below f16's smallest normal number, at a scale of the logits that makes them count."""
    K = deep(K, fmt)
    words, s, b, _ = table(V, K, fmt)
    rng = np.random.default_rng([8, M, K])
    tiny = lambda shape: (rng.integers(1, 1024, shape) * 2.0 ** -24).astype(np.float16)  # noqa: E731
    a = (tiny((M, K)) * rng.choice([-1, 1], (M, K))).astype(np.float16)
    s = np.where(rng.random(s.shape) < 0.5, tiny(s.shape), s).astype(np.float16)
    if b is not None:
        b = np.where(rng.random(b.shape) < 0.5, -tiny(b.shape), b).astype(np.float16)
    W = fr.mo.dequant(words, s, V, K, *fmt, b)
    scale = 2.0 ** 15
    targets = rng.integers(0, V, (M, 2)).astype(np.int32)
    compare(Call(handle(words, s, b, V, K, fmt), M, 0, 2, 5, scale, targets)(dev(a)), a, W, scale, targets, 5)
