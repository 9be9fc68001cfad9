"""Products with quantised weights whose results are never stored as they are: their plain forms and the framework's calls, and
the calls that are timed.

  product   out = residual + act(a W^T + bias), or residual + act(gate) * up of a weight that holds the gate's columns and
            then the up projection's; a f16 [M][K], bias f32, residual and out f16 or f32 with rows that may lie apart
  mlp       a layer's two in a row: silu(gate) * up in f16, then the down projection added to the f32 residual stream
  logprobs  logits = scale a W^T over a vocabulary table's first n_vocab rows: the log probabilities of given tokens, the
            entropy of each row's distribution, and the top_k tokens with theirs (largest first, equal ones by their number)

W [N][K] is quantised in blocks of 32 consecutive k of a row, `bits` u32 words each: 4 bits element e at bits 4 (e % 8) of
word e / 8; 2 bits at bits 2 (e % 16) of word e / 16; 3 bits the same and its third bit at bit e of word 2. One f16 scale s
(and, asymmetric, one f16 bias b) for each `group` values of a row: w = s (code - 2^(bits - 1)), asymmetric w = s code + b.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"
D, INNER, VOCAB = 2048, 6144, 248320  # the framework's model: hidden size, MLP width, rows of the embedding table
FORMATS = [(4, 32, False)] * 3 + [(4, 64, False), (4, 32, True), (3, 32, False), (3, 64, True), (2, 32, False), (2, 64, True)]


def _product(M, N, K, fmt=(4, 32, False), act="none", gated=False, bias=False, residual="none", out="f16", pad=0):
    return dict(kind="product", M=M, N=N, K=K, bits=fmt[0], group=fmt[1], asym=fmt[2], act=act, gated=gated, bias=bias,
                residual=residual, out=out, pad=pad)


def _mlp(M, hidden=D, inner=INNER):
    return dict(kind="mlp", M=M, D=hidden, I=inner)


def _logprobs(M, V, K, fmt=(4, 32, False), n_vocab=0, targets=1, top_k=0, scale=1.0):
    return dict(kind="logprobs", M=M, V=V, K=K, bits=fmt[0], group=fmt[1], asym=fmt[2], n_vocab=n_vocab or V, targets=targets,
                top_k=top_k, scale=scale)


def listed():
    return [
        # the MLP's first product of a single token: latency
        dict(_product(1, 2 * INNER, D, act="silu", gated=True), name="gated 1x12288x2048"),
        # the same for a long prompt: the matrix cores
        dict(_product(2048, 2 * INNER, D, act="silu", gated=True), name="gated 2048x12288x2048"),
        # the MLP's second product of a single token, onto the residual stream
        dict(_product(1, D, INNER, residual="f32", out="f32"), name="residual 1x2048x6144"),
        # an adapter's projection with its bias, rows apart, in another format, of a short prompt
        dict(_product(333, 2000, D, (3, 64, True), act="gelu", bias=True, residual="f16", pad=48), name="bias gelu residual 333x2000x2048"),
        # the MLP's second product of a long prompt
        dict(_product(2048, D, INNER, residual="f32", out="f32"), name="residual 2048x2048x6144"),
        # a layer's MLP in a small batch's decode step
        dict(_mlp(8), name="mlp 8"),
        # and for a question's rows behind a cached document
        dict(_mlp(61), name="mlp 61"),
        # the answer of one sequence: its label's probability and the alternatives
        dict(_logprobs(1, VOCAB, D, top_k=8), name="logprobs 1x248320"),
        # a decode step of a batch, four labels each, at a temperature
        dict(_logprobs(8, VOCAB, D, targets=4, top_k=20, scale=1.25), name="logprobs 8x248320"),
        # a question's tokens scored
        dict(_logprobs(61, VOCAB, D), name="logprobs 61x248320"),
        # a smaller vocabulary that is padded, in 3 bits
        dict(_logprobs(37, 151936, D, (3, 64, True), n_vocab=151669, targets=2, top_k=5), name="logprobs 37x151936 3-bit"),
        # a long prompt scored, with the alternatives of each position
        dict(_logprobs(2048, VOCAB, D, top_k=5), name="logprobs 2048x248320"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["product", "product", "product", "mlp", "logprobs", "logprobs"])
    M = rng.choice([1, _spread(rng, 2, 16), _spread(rng, 2, 300), _spread(rng, 64, 2048)])
    fmt = rng.choice(FORMATS)
    K = 64 * _spread(rng, 2, 96)
    if fmt[1] == 64 and rng.random() < 0.7:
        K = -(-K // 128) * 128
    elif fmt[1] == 32 and rng.random() < 0.1:
        K += 32  # a last half tile
    if kind == "mlp":
        return _mlp(M, 128 * _spread(rng, 2, 16), 128 * _spread(rng, 2, 48))
    if kind == "product":
        gated = rng.random() < 0.4
        N = 2 * _spread(rng, 8, INNER) if gated else _spread(rng, 1, 2 * INNER)
        return _product(M, N, K, fmt, rng.choice(["none", "silu", "gelu"]) if not gated else rng.choice(["silu", "silu", "gelu"]), gated,
                        rng.random() < 0.4, rng.choice(["none", "f16", "f32"]), rng.choice(["f16", "f32"]), rng.choice([0, 0, 8, 5]))
    K = min(K, 4096)
    V = _spread(rng, 1000, VOCAB)
    while M * V * K > 2048 * VOCAB * D:
        M //= 2
    return _logprobs(M, V, K, fmt, V - rng.choice([0, 0, rng.randrange(1, 300)]), rng.randrange(1, 9), rng.choice([0, 1, 5, 20, 32]),
                     rng.choice([1.0, 1.0, 0.7, 1.5]))


# ---- inputs ----

def _weight(N, K, bits, group, asym, std, g):
    """Packed random codes [N][K / 32][bits], scales and biases of weights with about the standard deviation std."""
    q = torch.empty(N, K // 32, bits * 4, device=DEV, dtype=torch.uint8)
    q.random_(0, 256, generator=g)
    step = std / math.sqrt((4 ** bits - 1) / 12)
    s = (step * (0.6 + 0.8 * torch.rand(N, K // group, device=DEV, generator=g))).half()
    b = None
    if asym:
        b = (s.float() * (0.4 * torch.rand(N, K // group, device=DEV, generator=g) - (2 ** bits - 1) / 2)).half()
    return {"N": N, "K": K, "bits": bits, "group": group, "asym": asym, "q": q.view(torch.int32), "s": s, "b": b}


def _rows(M, N, dtype, pad, g, scale):
    """[M][N] values ~N(0, scale^2) in rows that lie N + pad apart."""
    t = torch.zeros(M, N + pad, device=DEV, dtype=dtype)
    t[:, :N] = scale * torch.randn(M, N, device=DEV, generator=g)
    return t[:, :N]


def _middle(M, K, g):
    """What a gated activation leaves: many small values, some large."""
    x = torch.randn(M, K, device=DEV, generator=g)
    return (x * torch.sigmoid(x) * torch.randn(M, K, device=DEV, generator=g)).half()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + 29)
    M, st = case["M"], {"case": case}
    if case["kind"] == "product":
        N, K = case["N"], case["K"]
        cols = N // 2 if case["gated"] else N
        st["w"] = _weight(N, K, case["bits"], case["group"], case["asym"], 1 / math.sqrt(K), g)
        st["a"] = (torch.randn(M, K, device=DEV, generator=g) if case["gated"] else _middle(M, K, g) * 2).half().contiguous()
        st["bias"] = 0.5 * torch.randn(N, device=DEV, generator=g) if case["bias"] else None
        st["res"] = None
        if case["residual"] != "none":
            st["res"] = _rows(M, cols, torch.float32 if case["residual"] == "f32" else torch.float16, case["pad"], g, 2.0)
        st["out"] = _rows(M, cols, torch.float32 if case["out"] == "f32" else torch.float16, case["pad"], g, 0.0)
    elif case["kind"] == "mlp":
        H, I = case["D"], case["I"]
        st["up"] = _weight(2 * I, H, 4, 32, False, 1 / math.sqrt(H), g)
        st["down"] = _weight(H, I, 4, 32, False, 1 / math.sqrt(I), g)
        st["a"] = torch.randn(M, H, device=DEV, generator=g).half()
        st["x"] = 2.0 * torch.randn(M, H, device=DEV, generator=g)
        st["mid"] = torch.empty(M, I, device=DEV, dtype=torch.float16)
        st["out"] = torch.empty(M, H, device=DEV)
    else:
        V, K, n = case["V"], case["K"], case["n_vocab"]
        st["w"] = w = _weight(V, K, case["bits"], case["group"], case["asym"], 2 / math.sqrt(K), g)
        # normed rows that lean to a token, from not at all to near certainty; it is the first target of half of them
        t = torch.randint(0, n, (M,), device=DEV, generator=g)
        lean = 5.0 * torch.rand(M, 1, device=DEV, generator=g)
        st["a"] = (torch.randn(M, K, device=DEV, generator=g) + lean * _dense(w, t)).half()
        targets = torch.randint(0, n, (M, case["targets"]), device=DEV, generator=g)
        targets[::2, 0] = t[::2]
        st["targets"] = targets.int()
        st["logp"] = torch.empty(M, case["targets"], device=DEV)
        st["entropy"] = torch.empty(M, device=DEV)
        st["top_ids"] = torch.empty(M, case["top_k"], device=DEV, dtype=torch.int32)
        st["top_logp"] = torch.empty(M, case["top_k"], device=DEV)
    if own:
        _own_state(st)
    torch.cuda.synchronize()
    return st


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "strands-decider-web_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import hybrid_attention
    return hybrid_attention


def _own_state(st):
    """The handles, descriptions and workspace that a program keeps beside its data."""
    ha, case = _framework(), st["case"]

    def handle(w):
        return ha.MnbWeight(w["N"], w["K"], w["q"], w["s"], w["b"], bits=w["bits"], group=w["group"], asym=w["asym"])

    def code(t):
        return ha.F32 if t.dtype == torch.float32 else ha.F16

    if case["kind"] == "product":
        st["h"] = handle(st["w"])
        r, o = st["res"], st["out"]
        kw = {} if r is None else dict(residual=r, residual_dtype=code(r), residual_stride=r.stride(0))
        st["ep"] = ha.Epilogue(act=case["act"], gated=case["gated"], bias=st["bias"], out_dtype=code(o), out_stride=o.stride(0), **kw)
    elif case["kind"] == "mlp":
        st["h_up"], st["h_down"] = handle(st["up"]), handle(st["down"])
        st["ep_up"] = ha.Epilogue(act="silu", gated=True)
        st["ep_down"] = ha.Epilogue(residual=st["x"], residual_dtype=ha.F32, out_dtype=ha.F32)
    else:
        st["h"] = handle(st["w"])
        k = case["top_k"]
        st["lp"] = ha.LogProbs(n_vocab=case["n_vocab"], scale=case["scale"], targets=st["targets"], n_targets=case["targets"], top_k=k,
                               logp=st["logp"], entropy=st["entropy"], top_ids=st["top_ids"] if k else None,
                               top_logp=st["top_logp"] if k else None)
        st["ws"] = torch.empty(st["h"].logprobs_bytes(case["M"], st["lp"]), device=DEV, dtype=torch.uint8)


# ---- the operators in plain form ----

def _dense(w, rows=slice(None), dtype=torch.float32):
    """Weight rows as the numbers they stand for."""
    q, s = w["q"][rows], w["s"][rows].to(dtype)
    e = torch.arange(32, device=DEV, dtype=torch.int32)
    if w["bits"] == 4:
        c = (q[..., None] >> (4 * e[:8])) & 15
    else:
        c = ((q[..., :2, None] >> (2 * e[:16])) & 3)
        if w["bits"] == 3:
            c = c.flatten(-2) + 4 * ((q[..., 2:] >> e) & 1)
    c = c.reshape(q.shape[0], -1, w["group"]).to(dtype)
    if w["asym"]:
        return (c * s[..., None] + w["b"][rows].to(dtype)[..., None]).flatten(1)
    return ((c - 2 ** (w["bits"] - 1)) * s[..., None]).flatten(1)


def _times(a, w, dtype=torch.float32):
    return torch.matmul(a.to(dtype), _dense(w, dtype=dtype).T.contiguous())


def _act(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":  # the tanh form
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _fused(a, w, act, gated, bias, res):
    z = _times(a, w)
    if bias is not None:
        z = z + bias
    half = w["N"] // 2
    z = _act(z[:, :half], act) * z[:, half:] if gated else _act(z, act)
    return z if res is None else res.float() + z


def _log_probs(st):
    # in 64 bits: the order of two tokens can hang on the last digits, and so does the logarithm of a probability near one
    case, k, n = st["case"], st["case"]["top_k"], st["case"]["n_vocab"]
    z = case["scale"] * _times(st["a"], st["w"], torch.float64)[:, :n]
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1)
    lse = total.log()
    out = {"logp": (z.gather(1, st["targets"].long()) - lse[:, None]).float(), "entropy": (lse - (e * z).sum(-1) / total).float()}
    if k:
        ids = z.topk(min(n, k + 8), -1).indices.sort(-1).values
        top = z.gather(1, ids).sort(dim=-1, descending=True, stable=True)  # equal ones by their number
        out["top_ids"] = ids.gather(1, top.indices)[:, :k].int()
        out["top_logp"] = (top.values[:, :k] - lse[:, None]).float()
    return out


def run(st):
    case = st["case"]
    M = case["M"]
    if own:
        if case["kind"] == "product":
            st["h"].fused(M, st["a"], st["out"], st["ep"])
            return {"out": st["out"]}
        if case["kind"] == "mlp":
            st["h_up"].fused(M, st["a"], st["mid"], st["ep_up"])
            st["h_down"].fused(M, st["mid"], st["out"], st["ep_down"])
            return {"mid": st["mid"], "out": st["out"]}
        st["h"].logprobs(M, st["a"], st["lp"], st["ws"])
        return {name: st[name] for name in ("logp", "entropy", "top_ids", "top_logp")[:4 if case["top_k"] else 2]}
    if case["kind"] == "product":
        return {"out": _fused(st["a"], st["w"], case["act"], case["gated"], st["bias"], st["res"]).to(st["out"].dtype)}
    if case["kind"] == "mlp":
        mid = _fused(st["a"], st["up"], "silu", True, None, None).half()
        return {"mid": mid, "out": _fused(mid, st["down"], "none", False, None, st["x"])}
    return _log_probs(st)


# ---- what a pass cannot do without ----

def work(case):
    M = case["M"]
    if case["kind"] == "mlp":
        H, I = case["D"], case["I"]
        return {"bytes": 3 * H * I * 9 // 16 + M * (H * 2 + I * 4 + H * 8), "flops": 6 * M * H * I}
    N, K = case["V" if case["kind"] == "logprobs" else "N"], case["K"]
    n = case.get("n_vocab", N)
    b = n * (K // 32 * 4 * case["bits"] + K // case["group"] * (4 if case["asym"] else 2)) + M * K * 2
    if case["kind"] == "logprobs":
        return {"bytes": b + M * (8 * case["targets"] + 4 + 8 * case["top_k"]), "flops": 2 * M * n * K}
    size = {"none": 0, "f16": 2, "f32": 4}
    cols = N // 2 if case["gated"] else N
    return {"bytes": b + M * cols * (size[case["out"]] + size[case["residual"]]) + (4 * N if case["bias"] else 0),
            "flops": 2 * M * N * K}


# ---- the same in 64 bits, from the bytes ----

def _weight64(w, lo, hi):
    """Rows lo .. hi - 1 of the weight: each bit of a code by itself."""
    raw = w["q"][lo:hi].contiguous().view(torch.uint8)  # [rows][blocks][4 bits]
    k = torch.arange(32, device=DEV)
    if w["bits"] == 4:
        code = (raw[..., k // 2] // torch.where(k % 2 == 1, 16, 1)) % 16
    else:
        code = (raw[..., k // 4] // 4 ** (k % 4)) % 4
        if w["bits"] == 3:
            code = code + 4 * ((raw[..., 8 + k // 8] // 2 ** (k % 8)) % 2)
    code = code.double().flatten(1)
    at = torch.arange(w["K"], device=DEV) // w["group"]
    s = w["s"][lo:hi].double()[:, at]
    return code * s + w["b"][lo:hi].double()[:, at] if w["asym"] else (code - 2.0 ** (w["bits"] - 1)) * s


def _product64(a, w):
    y = torch.empty(a.shape[0], w["N"], dtype=torch.float64, device=DEV)
    for n in range(0, w["N"], 8192):
        y[:, n:n + 8192] = a.double() @ _weight64(w, n, min(w["N"], n + 8192)).T.contiguous()
    return y


def _act64(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "mlp":
        I = case["I"]
        z = _product64(st["a"], st["up"])
        mid = _act64(z[:, :I], "silu") * z[:, I:]
        # the second product's input is the first one's f16 output, and which way its values round is not its matter
        return {"mid": mid, "out": st["x"].double() + _product64(mid.half(), st["down"])}
    if case["kind"] == "product":
        z = _product64(st["a"], st["w"])
        if case["bias"]:
            z += st["bias"].double()
        if case["gated"]:
            z = _act64(z[:, :case["N"] // 2], case["act"]) * z[:, case["N"] // 2:]
        else:
            z = _act64(z, case["act"])
        return {"out": z if st["res"] is None else z + st["res"].double()}
    n, k = case["n_vocab"], case["top_k"]
    res = {name: [] for name in ("logp", "entropy", "top_ids", "top_logp")[:4 if k else 2]}
    for r in range(0, case["M"], 512):
        lp = torch.log_softmax(case["scale"] * _product64(st["a"][r:r + 512], st["w"])[:, :n], -1)
        res["logp"].append(lp.gather(1, st["targets"][r:r + 512].long()))
        res["entropy"].append(-(lp.exp() * lp).sum(-1))
        if k:
            top = lp.topk(k, -1)
            res["top_logp"].append(top.values)
            res["top_ids"].append(top.indices.int())
    return {name: torch.cat(v) for name, v in res.items()}
