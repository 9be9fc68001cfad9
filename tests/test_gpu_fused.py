"""Products with their bias, activation and residual (ha_mnb_fused) against 64 bits: every format, results of both types, odd
sizes from one row and column to many, strides, in place, streams and captured graphs."""
import numpy as np
import pytest

import fused_ref as fr
import hybrid_attention as ha

pytestmark = pytest.mark.gpu
FORMATS = [(4, 32, False), (4, 64, False), (4, 32, True), (4, 64, True), (3, 32, False), (3, 64, True), (2, 32, True), (2, 64, False)]
NP = {ha.F32: np.float32, ha.F16: np.float16}
DEV = "cuda:0"


def dev(x):
    import torch
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x.view(np.int32) if x.dtype == np.uint32 else x)).to(DEV)


def handle(words, s, b, N, K, fmt):
    return ha.MnbWeight(N, K, dev(words), dev(s), dev(b), bits=fmt[0], group=fmt[1], asym=fmt[2])


def check(got, want, off, K, dtype):
    """got (f64) against want: within the f32 arithmetic's `off` and the last rounding; f32 results in the norm too."""
    half = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 if dtype == ha.F16 else 0.0
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) - off - half).max()
    assert worst <= 0, "%.3g beyond the bound" % worst
    if dtype == ha.F32:
        rel = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
        assert rel <= 3 * fr.norm_tol(K) + 2.0 ** -23, "%.3g of the norm" % rel  # (3: gated products, activations)


def run(M, N, K, fmt=(4, 32, False), act=None, gated=False, bias=False, residual=None, out=ha.F16, pad=0, inplace=False, seed=0):
    import torch
    words, s, b, W = fr.weight(N, K, *fmt, seed=seed)
    rng = np.random.default_rng([seed, M, N, K])
    a = rng.standard_normal((M, K)).astype(np.float16)
    cols = N // 2 if gated else N
    bv = rng.standard_normal(N).astype(np.float32) if bias else None
    r = None if residual is None else (2 * rng.standard_normal((M, cols + pad))).astype(NP[residual])
    w = handle(words, s, b, N, K, fmt)
    rd = dev(r)
    od = rd if inplace else torch.full((M, cols + pad), 777.0, device=DEV, dtype=torch.float32 if out == ha.F32 else torch.float16)
    e = ha.Epilogue(act=act, gated=gated, bias=dev(bv), residual=rd, residual_dtype=out if residual is None else residual,
                    residual_stride=cols + pad, out_dtype=out, out_stride=cols + pad)
    w.fused(M, dev(a), od, e)
    torch.cuda.synchronize()
    got = od.cpu().numpy()
    if pad:
        assert (got[:, cols:] == (r[:, cols:] if inplace else 777.0)).all()
    want, off = fr.fused(a, W, act, gated, bv, None if r is None else r[:, :cols])
    check(got[:, :cols].astype(np.float64), want, off, K, out)
    w.close()
    return got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 256, 512), (5, 96, 256), (16, 64, 128), (33, 160, 384), (70, 320, 2048), (300, 272, 512)])
def test_formats(fmt, M, N, K):
    run(M, N, K, fmt, out=ha.F32)
    run(M, N, K, fmt, act="silu", gated=True, bias=True, seed=1)


@pytest.mark.parametrize("M", [1, 2, 3, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 128, 129, 200, 255, 257, 511, 640])
def test_rows(M):
    run(M, 512, 512, out=ha.F32, residual=ha.F32)
    run(M, 512, 512, act="silu", gated=True)


@pytest.mark.parametrize("N", [1, 2, 7, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 250, 255, 258, 511, 1000, 2049])
@pytest.mark.parametrize("M", [1, 20, 150, 400])
def test_columns(N, M):
    run(M, N, 192, residual=ha.F16, out=ha.F32, bias=True)
    if N % 2 == 0:
        run(M, N, 192, act="gelu", gated=True, bias=True, residual=ha.F32)


@pytest.mark.parametrize("K", [32, 64, 96, 128, 160, 192, 256, 320, 448, 576, 1024, 2080, 4096, 6144])
@pytest.mark.parametrize("M", [1, 4, 60, 300])
def test_depths(K, M):
    run(M, 144, K, out=ha.F32)
    if K % 64 == 0:
        run(M, 144, K, (3, 64, True), out=ha.F32)


@pytest.mark.parametrize("M,N,K", [(1, 12288, 2048), (61, 12288, 2048), (300, 12288, 2048)])
def test_gate_up(M, N, K):
    run(M, N, K, act="silu", gated=True)


@pytest.mark.parametrize("M,N,K", [(1, 2048, 6144), (61, 2048, 6144), (257, 2048, 6144), (130, 8256, 2048)])
def test_residual_stream(M, N, K):
    run(M, N, K, residual=ha.F32, out=ha.F32, inplace=True)


@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("out,residual", [(ha.F16, ha.F16), (ha.F16, ha.F32), (ha.F32, ha.F16), (ha.F32, None)])
@pytest.mark.parametrize("M", [3, 90, 300])
def test_strides(M, out, residual, pad):
    run(M, 200, 256, act="gelu", bias=True, residual=residual, out=out, pad=pad)


@pytest.mark.parametrize("dtype", [ha.F16, ha.F32])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_in_place(M, dtype):
    run(M, 260, 512, act="silu", gated=True, residual=dtype, out=dtype, pad=6, inplace=True)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_unaligned_weights(M):
    """Codes, scales and biases off the alignment that the fast kernels need."""
    import torch
    for fmt in [(4, 32, False), (3, 32, True), (2, 64, True)]:
        N, K = 100, 256
        words, s, b, W = fr.weight(N, K, *fmt, seed=3)
        a = np.random.default_rng(M).standard_normal((M, K)).astype(np.float16)
        q = torch.zeros(words.size + 1, dtype=torch.int32, device=DEV)
        q[1:] = dev(words).flatten()
        sd, bd = (torch.zeros(s.size + 1, dtype=torch.float16, device=DEV) for _ in range(2))
        sd[1:] = dev(s).flatten()
        if fmt[2]:
            bd[1:] = dev(b).flatten()
        w = ha.MnbWeight(N, K, q[1:], sd[1:], bd[1:] if fmt[2] else None, bits=fmt[0], group=fmt[1], asym=fmt[2])
        out = torch.empty(M, N, device=DEV)
        w.fused(M, dev(a), out, ha.Epilogue(out_dtype=ha.F32))
        torch.cuda.synchronize()
        want, off = fr.fused(a, W)
        check(out.cpu().numpy().astype(np.float64), want, off, K, ha.F32)


@pytest.mark.parametrize("M", [1, 17, 300])
def test_values(M):
    """Large and small inputs: saturated gates, f16 overflow to infinity, and a NaN or infinity in one row stays in it."""
    import torch
    N, K = 128, 256
    words, s, b, W = fr.weight(N, K, seed=5, std=4.0)
    w = handle(words, s, b, N, K, (4, 32, False))
    a = np.random.default_rng(6).standard_normal((M, K)).astype(np.float16)
    out = torch.empty(M, N // 2, device=DEV)
    w.fused(M, dev(a), out, ha.Epilogue(act="silu", gated=True, out_dtype=ha.F32))
    torch.cuda.synchronize()
    want, off = fr.fused(a, W, "silu", True)
    got = out.cpu().numpy().astype(np.float64)
    assert (np.abs(got - want) <= off + 2.0 ** -20 * 120 * np.abs(want) + 1e-37).all()  # (2^-24 of an argument up to 1000 in exp)
    big = (a.astype(np.float32) * 3000).astype(np.float16)
    o16 = torch.empty(M, N, device=DEV, dtype=torch.float16)
    w.fused(M, dev(big), o16, ha.Epilogue())
    torch.cuda.synchronize()
    z = big.astype(np.float64) @ W.T
    got = o16.cpu().numpy()
    assert (np.isinf(got) == (np.abs(z) >= 65520)).all() and (np.sign(got) == np.sign(z)).all()
    if M > 1:
        bad = a.copy()
        bad[1, 7], bad[M - 1, 100] = np.nan, np.inf
        w.fused(M, dev(bad), o16, ha.Epilogue())
        torch.cuda.synchronize()
        fine = np.isfinite(o16.cpu().numpy())
        assert not fine[1].any() and not fine[M - 1].any() and fine[[m for m in range(M) if m not in (1, M - 1)]].all()


def test_rows_do_not_touch_others():
    """Rows behind the last and columns behind the last are left as they were."""
    import torch
    for M, N in [(1, 20), (17, 100), (130, 130), (300, 300)]:
        words, s, b, W = fr.weight(N, 128, seed=8)
        a = np.random.default_rng(9).standard_normal((M + 40, 128)).astype(np.float16)
        buf = torch.full((M + 40, N + 30), 5.0, device=DEV)
        w = handle(words, s, b, N, 128, (4, 32, False))
        w.fused(M, dev(a), buf, ha.Epilogue(out_dtype=ha.F32, out_stride=N + 30))
        torch.cuda.synchronize()
        assert (buf[M:] == 5.0).all() and (buf[:, N:] == 5.0).all()


@pytest.mark.parametrize("M", [1, 61, 300])
def test_same_bits_on_a_stream_and_in_a_graph(M):
    import torch
    N, K = 640, 512
    words, s, b, W = fr.weight(N, K, seed=11)
    w = handle(words, s, b, N, K, (4, 32, False))
    a = torch.randn(M, K, device=DEV).half()
    first = torch.empty(M, N // 2, device=DEV, dtype=torch.float16)
    e = ha.Epilogue(act="silu", gated=True)
    torch.cuda.synchronize()
    w.fused(M, a, first, e)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    o2, o3 = torch.zeros_like(first), torch.zeros_like(first)
    torch.cuda.synchronize()
    w.fused(M, a, o2, e, stream=st.cuda_stream)
    st.synchronize()
    assert torch.equal(o2, first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.fused(M, a, o3, e, stream=torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        o3.zero_()
        a.copy_(torch.randn(M, K, device=DEV).half())
        g.replay()
        torch.cuda.synchronize()
        w.fused(M, a, first, e)
        torch.cuda.synchronize()
        assert torch.equal(o3, first), k


def test_a_run_of_calls():
    """A layer's MLP on the residual stream with its norm, as a host queues it, against 64 bits on the values each step stored."""
    import torch
    M, D, I = 37, 256, 384
    up, down = fr.weight(2 * I, D, seed=20), fr.weight(D, I, seed=21)
    wu, wd = handle(*up[:3], 2 * I, D, (4, 32, False)), handle(*down[:3], D, I, (4, 32, False))
    rng = np.random.default_rng(22)
    x0 = rng.standard_normal((M, D)).astype(np.float32)
    x, norm = dev(x0), torch.ones(D, device=DEV)
    h, mid = torch.empty(M, D, device=DEV, dtype=torch.float16), torch.empty(M, I, device=DEV, dtype=torch.float16)
    eu, ed = ha.Epilogue(act="silu", gated=True), ha.Epilogue(residual=x, out_dtype=ha.F32)
    for _ in range(3):
        before = x.cpu().numpy()
        torch.cuda.synchronize()
        ha.add_norm(M, D, M, x, None, norm, h)
        wu.fused(M, h, mid, eu)
        wd.fused(M, mid, x, ed)
        torch.cuda.synchronize()
        want, off = fr.fused(h.cpu().numpy(), up[3], "silu", True)
        check(mid.cpu().numpy().astype(np.float64), want, off, D, ha.F16)
        want, off = fr.fused(mid.cpu().numpy(), down[3], residual=before)
        check(x.cpu().numpy().astype(np.float64), want, off, I, ha.F32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 2])
@pytest.mark.parametrize("N,K", [(6, 64), (130, 1984), (34, 2112), (1022, 4160), (16, 16384), (16, 32768)])
def test_one_and_two_rows(M, fmt, N, K):
    """Lanes without a block, blocks in one to eight steps, columns past the last; rows longer than go through LDS."""
    if fmt[1] == 64 and K % 64:
        pytest.skip("K is not whole groups")
    run(M, N, K, fmt, out=ha.F32, bias=True, residual=ha.F16, pad=3)
    run(M, N, K, fmt, act="gelu", gated=True, bias=True, residual=ha.F32, out=ha.F32, pad=1, inplace=True)


@pytest.mark.parametrize("fmt", [(4, 32, True), (3, 32, False), (2, 32, True)])
@pytest.mark.parametrize("M", [1, 2, 3])
def test_operands_at_odd_places(M, fmt):
    """Codes 4 bytes and scales 2 bytes past an aligned address, one to three rows of an odd number of blocks."""
    import torch
    N, K = 50, 32 * 67
    words, s, b, W = fr.weight(N, K, *fmt, seed=4)
    a = np.random.default_rng(M).standard_normal((M, K)).astype(np.float16)

    def late(x, by):
        raw = torch.from_numpy(np.concatenate([np.zeros(by, np.uint8), np.ascontiguousarray(x).view(np.uint8).ravel()])).to(DEV)
        assert raw.data_ptr() % 16 == 0
        return raw, raw.data_ptr() + by
    q, sd, bd = late(words, 4), late(s, 2), None if b is None else late(b, 2)
    w = ha.MnbWeight(N, K, q[1], sd[1], bd and bd[1], bits=fmt[0], group=fmt[1], asym=fmt[2])
    out = torch.empty(M, N, device=DEV)
    w.fused(M, dev(a), out, ha.Epilogue(out_dtype=ha.F32))
    torch.cuda.synchronize()
    want, off = fr.fused(a, W)
    check(out.cpu().numpy().astype(np.float64), want, off, K, ha.F32)
    w.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1000, 2048, 2048), (1024, 1999, 4096)])
def test_halves_of_k(M, fmt, N, K):
    """Many rows of few columns: waves that take half of K each and finish half of the row tiles each."""
    run(M, N, K, fmt, out=ha.F32, bias=True, residual=ha.F32, inplace=True, pad=5)
    run(M, N, K, fmt, act="gelu", residual=ha.F16)


@pytest.mark.parametrize("M", [65, 96, 97, 192, 270, 333, 380])
def test_tiles_of_96_rows(M):
    run(M, 12288, 256, act="silu", gated=True, out=ha.F32)
    run(M, 5120, 512, (4, 32, True), out=ha.F32, bias=True)
    run(M, 5120, 512, (3, 64, False), residual=ha.F16)
