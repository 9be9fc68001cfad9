"""Products with what follows them (ha_mnb_fused) by every kernel and tile shape there is, in every format, against 64 bits: few and
many steps of K, plain and gated. tests/test_fused_coverage.py checks that the sizes here reach all of them."""
import numpy as np
import pytest

import hybrid_attention as ha
import test_gpu_fused as tf

pytestmark = pytest.mark.gpu
FORMATS = [(bits, group, asym) for bits in (4, 3, 2) for group in (32, 64) for asym in (False, True)]
# rows, rows of the weight, K, gated
SHALLOW = [(1, 26, 128, False), (1, 26, 128, True), (2, 26, 128, False), (2, 26, 128, True), (5, 26, 96, False), (5, 26, 96, True),
           (5, 26, 128, False), (5, 26, 128, True), (5, 26, 192, False), (5, 26, 192, True), (512, 12290, 128, False), (640, 100, 128, False),
           (640, 100, 128, True), (640, 202, 128, False), (640, 202, 128, True), (640, 398, 128, False), (640, 398, 128, True),
           (640, 998, 128, False), (640, 998, 128, True), (640, 998, 384, False), (700, 398, 128, False), (700, 398, 128, True),
           (1000, 202, 128, False), (1000, 202, 128, True), (1000, 398, 128, False), (1000, 398, 128, True), (1000, 998, 128, False),
           (1000, 998, 128, True), (1000, 998, 384, False), (1000, 4098, 128, False), (1000, 4098, 128, True), (1000, 12290, 128, True),
           (1000, 15998, 128, False), (1100, 100, 128, False), (1100, 100, 128, True), (1100, 202, 128, False), (1100, 202, 128, True),
           (1100, 998, 128, False), (1100, 1998, 128, False), (1100, 1998, 128, True)]
DEEP = [(1, 26, 1088, False), (2, 26, 1088, False), (5, 26, 1088, False), (5, 26, 1152, False), (5, 26, 4096, False), (5, 4098, 1152, False),
        (45, 4098, 1152, False), (160, 3002, 1152, False), (512, 12290, 1152, False), (640, 100, 1152, False), (640, 202, 1152, False),
        (640, 398, 1152, False), (640, 998, 1152, False), (640, 4098, 1152, True), (700, 398, 1152, False), (1000, 202, 1152, False),
        (1000, 398, 1152, False), (1000, 998, 1152, False), (1000, 1998, 1152, False), (1000, 1998, 4096, False), (1000, 4098, 1152, False),
        (1000, 12290, 1152, False), (1100, 1998, 1152, False)]


def in_formats(sizes):
    return [(M, N, K, fmt, gated) for M, N, K, gated in sizes for fmt in FORMATS if K % fmt[1] == 0]


def cases():
    return in_formats(SHALLOW + DEEP)


@pytest.mark.parametrize("M,N,K,fmt,gated", in_formats(SHALLOW))
def test_shallow(M, N, K, fmt, gated):
    tf.run(M, N, K, fmt, act="silu" if gated else None, gated=gated, bias=True, residual=ha.F32, out=ha.F32, pad=3, inplace=True)


@pytest.mark.parametrize("M,N,K,fmt,gated", in_formats(DEEP))
def test_deep(M, N, K, fmt, gated):
    tf.run(M, N, K, fmt, act="gelu" if gated else None, gated=gated, out=ha.F32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 90, 256), (2, 90, 256), (5, 90, 256), (5, 90, 192), (640, 398, 128), (1000, 4098, 128), (512, 12290, 128)])
def test_subnormal_operands(M, N, K, fmt):
    """Values of a, scales and biases below f16's smallest normal number, 2^-14, count as they are, in dot products of the vector unit
    and on the matrix unit alike."""
    import torch
    import fused_ref as fr
    bits, group, asym = fmt
    words, s, b, _ = fr.weight(N, K, *fmt, seed=60)
    rng = np.random.default_rng([61, M, N, K])
    tiny = lambda shape: (rng.integers(1, 1024, shape) * 2.0 ** -24).astype(np.float16)  # noqa: E731
    a = np.where(rng.random((M, K)) < 0.7, tiny((M, K)) * rng.choice([-1, 1], (M, K)), rng.standard_normal((M, K)) * 2.0 ** -10).astype(np.float16)
    a[0] = tiny(K)  # (a row of nothing else)
    s = np.where(rng.random(s.shape) < 0.7, tiny(s.shape), s * np.float16(2.0 ** -9)).astype(np.float16)
    s[0] = tiny(K // group)
    if asym:
        b = np.where(rng.random(b.shape) < 0.7, -tiny(b.shape), b * np.float16(2.0 ** -9)).astype(np.float16)
    W = fr.mo.dequant(words, s, N, K, *fmt, b)
    w = tf.handle(words, s, b, N, K, fmt)
    out = torch.empty(M, N, device=tf.DEV)
    w.fused(M, tf.dev(a), out, ha.Epilogue(out_dtype=ha.F32))
    torch.cuda.synchronize()
    want, off = fr.fused(a, W)
    got = out.cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all() and (np.abs(got - want) <= off).all()
    w.close()
