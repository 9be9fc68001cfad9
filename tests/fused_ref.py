"""Plain forms in 64 bits of the products whose results are not stored as they are, and how far f32 sums may be off them.

A sum of K products of f16 with exact weights is made of G = K / 32 group sums, each scaled and added in f32. Each addition is off
by at most half a step, 2^-24 of the partial sum. As independent errors that comes to about sqrt(G / 2) 2^-24 / sqrt(3) of the
result's size (partial sums grow to it), and what the matrix unit rounds within a group adds a few steps of a group's sum:
NORM allows four times that of the rms over the result. The bound of a single value (each) takes every rounding at its worst: G
additions, G products and 40 within groups and reductions, 2^-23 of sum |a| |w|. Weights rounded to f16 would be off by
2^-12 / sqrt(3) of the result's size, 1.4e-4."""
import numpy as np

import mnb_oracle as mo


def weight(N, K, bits=4, group=32, asym=False, seed=0, std=None):
    """Packed random codes, scales and biases (f16) of weights of about std, and the weights (f64)."""
    rng = np.random.default_rng([seed, N, K, bits])
    std = std or 1 / np.sqrt(K)
    words = rng.integers(0, 2 ** 32, (N, K // 32, mo.words_per_block(bits)), dtype=np.uint64).astype(np.uint32)
    step = std / np.sqrt((4 ** bits - 1) / 12)
    s = (step * (0.6 + 0.8 * rng.random((N, K // group)))).astype(np.float16)
    b = None
    if asym:
        b = (s.astype(np.float64) * (0.4 * rng.random((N, K // group)) - (2 ** bits - 1) / 2)).astype(np.float16)
    return words, s, b, mo.dequant(words, s, N, K, bits, group, asym, b)


def norm_tol(K):
    return 4 * 2.0 ** -24 * np.sqrt(K / 32 / 6 + 4)


def each_tol(K):
    return (K / 32 * 2 + 40) * 2.0 ** -23


def act(z, name):
    if name == "silu":
        return z / (1 + np.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
    return z


def fused(a, W, name=None, gated=False, bias=None, residual=None, K=None):
    """The result and, for each value, how far f32 arithmetic may be off it: sums as above; an activation passes errors on by at
    most 1.13 and adds a few steps of its own (exp, 1/x: 2^-20 of it with arguments up to 16)."""
    a64 = a.astype(np.float64)
    z, size = a64 @ W.T, np.abs(a64) @ np.abs(W).T
    if bias is not None:
        z, size = z + bias, size + np.abs(bias)
    off = each_tol(W.shape[1]) * size
    if gated:
        h = W.shape[0] // 2
        g = act(z[:, :h], name)
        out = g * z[:, h:]
        off = (1.13 * off[:, :h] + 2.0 ** -20 * np.abs(g)) * np.abs(z[:, h:]) + off[:, h:] * (np.abs(g) + 1.13 * off[:, :h])
    else:
        out = act(z, name)
        off = 1.13 * off + 2.0 ** -20 * np.abs(out) if name else off
    if residual is not None:
        out = out + residual.astype(np.float64)
    return out, off + 2.0 ** -23 * np.abs(out)


def logprobs(a, W, scale=1.0, targets=None, k=0):
    """logp, entropy, lse, ids, top logp in 64 bits, and how far off logp (targets, top) and entropy may be: a row's largest
    logits are multiplied out in 64 bits, so what the sum over all is off by comes from the others, each off by `delta` (the
    bound above on the norm, three times for a single one) and by its exponential's 2^-20."""
    z = scale * (a.astype(np.float64) @ W.T)
    K = W.shape[1]
    m = z.max(1, keepdims=True)
    e = np.exp(z - m)
    total = e.sum(1, keepdims=True)
    lse = (m + np.log(total))[:, 0]
    p, x = e / total, z - m
    H = np.log(total[:, 0]) - (p * x).sum(1)
    size = scale * np.sqrt((a.astype(np.float64) ** 2).sum(1)) * np.sqrt((W ** 2).sum(1).max())
    delta = 3 * norm_tol(K) * size + 2.0 ** -20
    rest = np.maximum(0, 1 - p.max(1))
    out = {"entropy": H, "lse": lse, "off": rest * delta,
           "entropy_off": 2 * delta * (rest * (1 + H) - (p * x).sum(1)) + 2.0 ** -23 * np.abs(H)}
    if targets is not None:
        ok = (targets >= 0) & (targets < W.shape[0])
        out["logp"] = np.where(ok, np.take_along_axis(z, np.where(ok, targets, 0), 1), np.nan) - lse[:, None]
    if k:
        out["ids"] = np.argsort(-z, axis=1, kind="stable")[:, :k]
        out["top"] = np.take_along_axis(z, out["ids"], 1) - lse[:, None]
    return out
