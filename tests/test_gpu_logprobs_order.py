"""The order of the largest tokens where logits are small beside their terms: f32 sums are off by what the terms are, not by what is
left of them, so which tokens are multiplied out in 64 bits must go by the terms."""
import numpy as np
import pytest

import fused_ref as fr
from test_gpu_logprobs import Call, check, dev, handle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [3000, 33000])  # stored logits, records
@pytest.mark.parametrize("fmt", [(4, 32, False), (4, 32, True), (3, 32, False), (2, 32, True)])
@pytest.mark.parametrize("M,K", [(3, 96), (50, 96), (3, 256), (16, 512), (40, 128), (140, 192), (600, 128)])
def test_cancelled_terms(M, K, fmt, V):
    """Groups 0 and 1 cancel: their products are some thousand, off by 1e-4 in f32. Group 2 gives eight tokens 0.01 and a few steps of
    7.6e-6 more, two of them in one block of 64, and all others -1."""
    bits, _, asym = fmt
    words, s, b, _ = fr.weight(V, K, *fmt, seed=70)
    rng = np.random.default_rng([71, M, K])
    step = 30 / 2 ** bits
    s[:, 0] = step * (0.6 + 0.8 * rng.random(V))
    words[:, 1], s[:, 1] = words[:, 0], s[:, 0]
    mid = 2 ** (bits - 1)
    if asym:
        b[:, 0] = -(mid - 0.5) * s[:, 0]
        b[:, 1] = b[:, 0]
    code = lambda c: np.array({4: [0x11111111 * c] * 4, 3: [0x55555555 * (c & 3)] * 2 + [0xFFFFFFFF * (c >> 2)],  # noqa: E731
                               2: [0x55555555 * c] * 2}[bits], np.uint32)
    at = 640
    tokens = [at + 5, at + 40, 64 * 3 + 1, 64 * 5 + 9, 64 * 20, 64 * 30 + 63, 64 * 33 + 2, 64 * 40 + 7]
    words[:, 2], s[:, 2] = code(mid - 1), 1.0
    words[tokens, 2] = code(mid + 1)
    s[tokens, 2] = np.float16(0.01) + np.arange(8)[::-1].astype(np.float16) * np.float16(2.0 ** -17)
    if asym:
        b[:, 2] = -mid * s[:, 2].astype(np.float32)
    W = fr.mo.dequant(words, s, V, K, *fmt, b)
    a = np.zeros((M, K), np.float16)
    a[:, :32] = 100 * rng.standard_normal((M, 32))
    a[:, 32:64] = -a[:, :32]
    a[:, 64:96] = 2.0 ** -5
    got = Call(handle(words, s, b, V, K, fmt), M, 0, 0, 6)(dev(a))
    want = fr.logprobs(a, W, k=6)
    assert (want["ids"] == tokens[:6]).all()
    check(got, want, 0, 6)
