"""The paged cache of 4-bit keys and values: its operators in plain form and through the framework, and the calls that are timed.

  append  a batch's fused qkv rows: q and k normed for each head and rotated to their positions, q returned, k and v put
          into the sequences' pages in 4 bits (and returned as the values they stand for)
  attend  causal attention of a batch's query rows over their sequences' pages, gated
  step    both, as a layer calls them

A batch is ragged: rows of sequence b are row_start[b] .. row_start[b+1] - 1, its context is len[b] tokens with them, token t
stands in page table[b][t / page], slot t % page. One page of one layer, for each KV head, first of keys and then of values:
  codes   [page][HD / 2] bytes: channel c of a row is nibble 16 ((c % G) / 4) + 4 (c / G) + c % 4, G = HD / 4, low nibble first
  params  [page / 4][4 groups][scale, zero][4 tokens] f16: channel c of group c / G stands for scale (code - 8) + zero
"""
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda:0"
THETA, EPS = 1e7, 1e-6
# (query heads, KV heads, head dim, rotated dims): the framework's model, and other layouts the cache takes
MODEL = (8, 2, 256, 64)
HEADS = [MODEL, MODEL, MODEL, (16, 2, 128, 128), (32, 8, 128, 128), (4, 4, 128, 64), (10, 2, 256, 64), (16, 1, 256, 256), (5, 1, 128, 32)]


def _case(kind, seqs, heads=MODEL, page=64, gated=True, f32=False):
    """seqs: "n x (cached + new)" texts, joined by commas, in the batch's order."""
    return dict(kind=kind, seqs=seqs, HQ=heads[0], HK=heads[1], HD=heads[2], rot=heads[3], page=page, gated=gated, f32=f32)


def _seqs(case):
    out = []
    for part in case["seqs"].split(","):
        n, lens = part.split("x")
        p, l = lens.split("+")
        out += [(int(p), int(l))] * int(n)
    return out


def _ragged(n, lo, hi, new, seed):
    """n sequences of lengths spread over [lo, hi], one text."""
    k = max(1, n - 1)
    order = sorted(range(n), key=lambda i: (i * 7919 + seed) % 104729)
    return ",".join("1x%d+%d" % (round(lo * (hi / lo) ** (i / k)), new) for i in order)


def listed():
    return [
        # a decode step's new rows of a batch: latency
        dict(_case("append", "8x1536+1"), name="append 8x1536+1"),
        # a question put behind a cached state document, rows as the f32 path has them
        dict(_case("append", "1x1531+61", f32=True), name="append 1x1531+61 f32"),
        # a prefill of eight sequences
        dict(_case("append", "8x0+2048"), name="append 8x2048"),
        # one token of one sequence: the smallest call
        dict(_case("attend", "1x1531+1"), name="attend 1x1531+1"),
        # a decode step of the batch whose f16 form the framework's engine serves
        dict(_case("attend", "8x1536+1"), name="attend 8x1536+1"),
        # a serving batch of uneven lengths
        dict(_case("attend", _ragged(48, 37, 4095, 1, 3), page=16), name="attend 48 ragged +1"),
        # one token on a very long context: cache bandwidth
        dict(_case("attend", "1x131071+1"), name="attend 1x131071+1"),
        # a question's rows on the cached state
        dict(_case("attend", "1x1531+61"), name="attend 1x1531+61"),
        # prefills and decode steps in one batch, heads of 128 without a gate
        dict(_case("attend", "1x0+777,5x900+1,1x2000+130,3x333+1,1x64+300", (32, 8, 128, 128), 32, False), name="attend mixed hd128"),
        # the prefill of eight sequences
        dict(_case("attend", "8x0+2048"), name="attend 8x2048"),
        # a layer's step: the rows in, their attention out
        dict(_case("step", "8x1536+1"), name="step 8x1536+1"),
        # a layer of a prefill behind a cached prefix
        dict(_case("step", "2x1000+1000"), name="step 2x1000+1000"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "attend", "step"])
    form = rng.choice(["token", "token", "suffix", "prompt", "mixed"])
    if form == "token":
        n, new = _spread(rng, 1, 64), 1
        seqs = [(_spread(rng, 1, min(32768, 131072 // n)), new) for _ in range(n)]
    elif form == "suffix":
        seqs = [(_spread(rng, 16, 4000), _spread(rng, 2, 96)) for _ in range(_spread(rng, 1, 8))]
    elif form == "prompt":
        n = _spread(rng, 1, 6)
        seqs = [(0, _spread(rng, 1, 2047)) for _ in range(n)]
    else:
        seqs = [(_spread(rng, 1, 3000), 1 if rng.random() < 0.6 else _spread(rng, 2, 500)) for _ in range(_spread(rng, 2, 12))]
    heads = rng.choice(HEADS)
    if form in ("prompt", "mixed") and heads[0] * heads[2] > 2048:
        heads = MODEL
    return _case(kind, ",".join("1x%d+%d" % s for s in seqs), heads, rng.choice([16, 32, 64, 128]),
                 heads[2] == 256 or rng.random() < 0.5, kind != "attend" and rng.random() < 0.25)


# ---- inputs ----

def _quantise(x):
    """Codes 0..15 (as int32), scales and zeros (f16) of f32 values [..., HD], by groups of HD / 4 channels. Rounded step by
    step in f32, so that codes at a border between two do not depend on who computes them."""
    v = x.unflatten(-1, (4, -1))
    lo, hi = v.amin(-1), v.amax(-1)
    z = (lo + (hi - lo) * np.float32(8 / 15).item()).to(torch.float16)
    zf = z.float()
    s = torch.maximum((hi - zf) * np.float32(1 / 7).item(), (zf - lo) * 0.125).to(torch.float16)
    bad = ~(torch.isfinite(s) & torch.isfinite(z))
    s, z = s.masked_fill(bad, float("nan")), z.masked_fill(bad, 0.0)
    sf, zf = s.float()[..., None], z.float()[..., None]
    c = ((v - zf) / sf).round() + 8
    c = torch.where((sf > 0), c.clamp(0, 15), torch.full_like(c, 8)).to(torch.int32)
    return c.flatten(-2), s, z


def _pack(c):
    """Codes [..., HD] to the row's bytes [..., HD / 2]: channel (group g, 4 i + e) is nibble 16 i + 4 g + e."""
    n = c.unflatten(-1, (4, -1, 4)).transpose(-3, -2).flatten(-3)
    return (n[..., 0::2] | (n[..., 1::2] << 4)).to(torch.uint8)


def _unpack(b):
    """The codes [..., HD] of a row's bytes [..., HD / 2]."""
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    return n.unflatten(-1, (-1, 4, 4)).transpose(-3, -2).flatten(-3)


def _values(c, s, z):
    """What codes stand for, f32."""
    return (s.float()[..., None] * (c.float() - 8).unflatten(-1, (4, -1)) + z.float()[..., None]).flatten(-2)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + 17)
    rng = np.random.default_rng([int(seed), 18])
    seqs = _seqs(case)
    HQ, HK, HD, ps = case["HQ"], case["HK"], case["HD"], case["page"]
    B, T = len(seqs), sum(l for _, l in seqs)
    lens = [p + l for p, l in seqs]
    need = [-(-n // ps) for n in lens]
    width, n_pages = max(need), sum(need) + 3
    ids = rng.permutation(n_pages)
    table = np.full((B, width), -1, np.int32)  # behind a sequence's last page the table says nothing
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum([l for _, l in seqs])]).astype(np.int32)
    # the pool: every slot holds a token's values, keys as norms leave them, values ~N(0, 1)
    pool = torch.empty(n_pages, HK, 2, ps * (HD // 2 + 16), device=DEV, dtype=torch.uint8)
    for a in range(0, n_pages, 4096 // ps + 1):  # blocks of pages: the f32 values stay small
        p = pool[a:a + 4096 // ps + 1]
        c, s, z = _quantise(torch.randn(p.shape[0], HK, 2, ps, HD, device=DEV, generator=g))
        p[..., :ps * HD // 2] = _pack(c).flatten(-2)
        sz = torch.stack([s, z], -1).unflatten(3, (ps // 4, 4)).permute(0, 1, 2, 3, 5, 6, 4)
        p[..., ps * HD // 2:] = sz.flatten(3).contiguous().view(torch.uint8)
    stride = HQ * HD * (2 if case["gated"] else 1) + 2 * HK * HD
    rows = torch.empty(T, stride, device=DEV, dtype=torch.float32 if case["f32"] else torch.float16)
    for a in range(0, T, 2048):
        rows[a:a + 2048] = torch.randn(min(2048, T - a), stride, device=DEV, generator=g)
    q = torch.empty(T, HQ, HD, device=DEV, dtype=torch.float16)
    for a in range(0, T, 2048):
        q[a:a + 2048] = 1.2 * torch.randn(min(2048, T - a), HQ, HD, device=DEV, generator=g)
    norms = {n: (1 + 0.1 * rng.standard_normal(HD)).astype(np.float32) for n in ("q_norm", "k_norm")}
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    s = {"case": case, "pool": pool, "rows": rows, "q": q, "table": dev(table), "lens": dev(np.array(lens, np.int32)),
         "start": dev(start), "T": T, "B": B, "max_rows": max(l for _, l in seqs), "max_len": max(lens), "stride": stride,
         "seq_of": dev(np.repeat(np.arange(B), [l for _, l in seqs])),
         "at": dev(np.concatenate([np.arange(l) for _, l in seqs])),
         "q_norm": dev(norms["q_norm"]), "k_norm": dev(norms["k_norm"]),
         "values": torch.empty(T, 2, HK, HD, device=DEV, dtype=torch.float16),
         "out": torch.empty(T, HQ, HD, device=DEV, dtype=torch.float16)}
    if own:
        ha = _framework()
        s["kv"] = ha.PagedKV(pool, n_pages, page_size=ps, max_ctx=max(lens), HQ=HQ, HK=HK, HD=HD, rot_dim=case["rot"],
                             gated=case["gated"], dtype=ha.F32 if case["f32"] else ha.F16, rope_theta=THETA, eps=EPS)
        for n, v in norms.items():
            s["kv"].set_param(0, n, v)
        s["batch"] = ha.KVBatch(B, T, s["max_rows"], s["max_len"], s["start"], s["lens"], s["table"], width)
    torch.cuda.synchronize()
    return s


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "strands-decider-web_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import hybrid_attention
    return hybrid_attention


# ---- the operators in plain form ----

def _positions(s):
    """The position of each row: its sequence's length less the rows from it on."""
    seq = s["seq_of"]
    return (s["lens"][seq] - (s["start"][seq + 1] - s["start"][seq])).long() + s["at"]


def _norm_rotate(x, w, pos, rot):
    """x [T, heads, HD] normed with gain w and rotated at pos, in x's type."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    ang = pos.double()[:, None] * THETA ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    cos, sin = ang.cos().float().to(x.dtype)[:, None], ang.sin().float().to(x.dtype)[:, None]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _append(s):
    case = s["case"]
    HQ, HK, HD, ps, T = case["HQ"], case["HK"], case["HD"], case["page"], s["T"]
    pos = _positions(s)
    per = HD * (2 if case["gated"] else 1)
    q = s["rows"][:, :HQ * per].unflatten(-1, (HQ, per))[..., :HD].float()
    kv = s["rows"][:, HQ * per:].unflatten(-1, (2, HK, HD))
    q = _norm_rotate(q, s["q_norm"], pos, case["rot"]).to(torch.float16)
    # 64 bits: a key next to a border between two codes
    k = _norm_rotate(kv[:, 0].double(), s["k_norm"], pos, case["rot"]).float()
    c, sc, z = _quantise(torch.stack([k, kv[:, 1].float()], 1))
    page, slot = s["table"][s["seq_of"], pos // ps].long()[:, None], (pos % ps)[:, None]
    byte = torch.arange(HD // 2, device=DEV)[None]
    pool = s["pool"].permute(0, 3, 1, 2)  # [page][byte][head][k, v]
    pool[page, slot * (HD // 2) + byte] = _pack(c).permute(0, 3, 2, 1)
    half = torch.arange(8, device=DEV)[None]  # (group, scale or zero)
    par = s["pool"][..., ps * HD // 2:].view(torch.float16).permute(0, 3, 1, 2)
    par[page, ((slot // 4) * 8 + half) * 4 + slot % 4] = torch.stack([sc, z], -1).flatten(3).permute(0, 3, 2, 1)
    return q, _values(c, sc, z).to(torch.float16)


def _attend(s, q):
    case = s["case"]
    HQ, HK, HD, ps, B = case["HQ"], case["HK"], case["HD"], case["page"], s["B"]
    pages = s["pool"][s["table"].clamp(min=0).long()]  # [B][pages][HK][k, v][bytes]
    c = _unpack(pages[..., :ps * HD // 2].unflatten(-1, (ps, HD // 2)))
    sz = pages[..., ps * HD // 2:].contiguous().view(torch.float16).unflatten(-1, (ps // 4, 4, 2, 4))
    sz = sz.permute(0, 1, 2, 3, 4, 7, 5, 6).flatten(4, 5)  # [B][pages][HK][k, v][token][group][2]
    x = _values(c, sz[..., 0], sz[..., 1]).permute(3, 0, 2, 1, 4, 5).flatten(3, 4)  # [k, v][B][HK][token][HD]
    M, N = s["max_rows"], x.shape[3]
    new = s["start"][1:] - s["start"][:-1]
    row = torch.arange(M, device=DEV)
    qp = q[(s["start"][:-1, None] + row).clamp(max=s["T"] - 1).long()].float()  # [B][M][HQ][HD]
    qp = qp.unflatten(2, (HK, HQ // HK)).permute(0, 2, 3, 1, 4).flatten(2, 3)    # [B][HK][heads x M][HD]
    sc = torch.matmul(qp, x[0].transpose(-1, -2).contiguous()) * (1 / math.sqrt(HD))
    last = (s["lens"] - new)[:, None] + row  # the last key that each row sees
    see = torch.arange(N, device=DEV) <= torch.minimum(last, s["lens"][:, None] - 1)[..., None]
    sc = sc.unflatten(2, (HQ // HK, M)).masked_fill(~see[:, None, None], float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(p.flatten(2, 3), x[1]).unflatten(2, (HQ // HK, M)) / p.sum(-1)[..., None]
    o = o.flatten(1, 2)[s["seq_of"], :, s["at"]]  # [T][HQ][HD]
    if case["gated"]:
        gate = s["rows"][:, :HQ * 2 * HD].unflatten(-1, (HQ, 2, HD))[:, :, 1].float()
        o = o * torch.sigmoid(gate)
    return o.to(torch.float16)


def run(s):
    kind = s["case"]["kind"]
    if own:
        kv, rows, stride = s["kv"], s["rows"], s["stride"]
        if kind != "attend":
            kv.append(0, s["batch"], rows, stride, s["q"], s["values"])
        if kind != "append":
            kv.attention(0, s["batch"], s["q"], rows, stride, s["out"])
        return {"append": {"q": s["q"], "kv": s["values"]}, "attend": {"out": s["out"]},
                "step": {"q": s["q"], "kv": s["values"], "out": s["out"]}}[kind]
    if kind == "attend":
        return {"out": _attend(s, s["q"])}
    q, values = _append(s)
    return {"q": q, "kv": values} if kind == "append" else {"q": q, "kv": values, "out": _attend(s, q)}


# ---- what a pass cannot do without ----

def work(case):
    seqs = _seqs(case)
    HQ, HK, HD = case["HQ"], case["HK"], case["HD"]
    T, e = sum(l for _, l in seqs), 4 if case["f32"] else 2
    row = HK * 2 * (HD // 2 + 16)  # a token's bytes in the cache
    cached = sum(p + l for p, l in seqs) * row
    b = f = 0
    if case["kind"] != "attend":
        b += T * ((HQ + 2 * HK) * HD * e + HQ * HD * 2 + row + 2 * HK * HD * 2)
        f += T * (HQ + 2 * HK) * HD * 8
    if case["kind"] != "append":
        b += cached + T * HQ * HD * (4 + (e if case["gated"] else 0))
        f += 4 * HQ * HD * sum(l * p + l * (l + 1) // 2 for p, l in seqs)
    return {"bytes": b, "flops": f}


# ---- the same in 64 bits, one sequence and head at a time ----

def _prep64(x, w, pos, rot):
    x = x / torch.sqrt(x.pow(2).mean(1, keepdim=True) + EPS) * w.double()
    y = x.clone()
    for i in range(rot // 2):
        a = pos.double() / THETA ** (2 * i / rot)
        y[:, i] = x[:, i] * a.cos() - x[:, i + rot // 2] * a.sin()
        y[:, i + rot // 2] = x[:, i + rot // 2] * a.cos() + x[:, i] * a.sin()
    return y


def _held64(x):
    """What the cache holds of x [n][HD], as codes, scales and zeros of each group."""
    parts = []
    for v in x.chunk(4, 1):
        lo, hi = v.min(1).values, v.max(1).values
        z = (lo + (hi - lo) * 8 / 15).half().double()
        s = torch.maximum((hi - z) / 7, (z - lo) / 8).half().double()
        c = torch.clamp(torch.round((v - z[:, None]) / s[:, None].clamp(min=1e-30)), -8, 7)
        parts.append(s[:, None] * c + z[:, None])
    return torch.cat(parts, 1)


def _read64(s, b, n, h, which):
    """Keys (0) or values (1) of sequence b's tokens 0..n-1 and KV head h, from the pages."""
    ps, HD = s["case"]["page"], s["case"]["HD"]
    t = torch.arange(n, device=DEV)
    page, slot = s["table"][b][t // ps].long(), t % ps
    raw = s["pool"][page, h, which]  # [n][bytes]
    c = torch.arange(HD, device=DEV)
    nib = 16 * ((c % (HD // 4)) // 4) + 4 * (c // (HD // 4)) + c % 4
    byte = raw.gather(1, slot[:, None] * (HD // 2) + (nib // 2)[None])
    code = (byte.long() >> (4 * (nib % 2))) & 15
    par = raw[:, ps * HD // 2:].contiguous().view(torch.float16).double()
    k = (slot[:, None] // 4 * 4 + (c // (HD // 4))[None]) * 8 + slot[:, None] % 4
    return par.gather(1, k) * (code - 8).double() + par.gather(1, k + 4)


def exact(case, seed):
    seqs = _seqs(case)
    HQ, HK, HD, rot, kind = case["HQ"], case["HK"], case["HD"], case["rot"], case["kind"]
    s = prepare(case, seed)
    per = HD * (2 if case["gated"] else 1)
    T = s["T"]
    q = torch.empty(T, HQ, HD, dtype=torch.float64, device=DEV)
    kv = torch.empty(T, 2, HK, HD, dtype=torch.float64, device=DEV)
    out = torch.empty(T, HQ, HD, dtype=torch.float64, device=DEV)
    at = 0
    for b, (P, L) in enumerate(seqs):
        r = s["rows"][at:at + L].double()
        pos = torch.arange(P, P + L, device=DEV)
        if kind == "attend":
            q[at:at + L] = s["q"][at:at + L].double()
        else:
            for h in range(HQ):
                q[at:at + L, h] = _prep64(r[:, h * per:h * per + HD], s["q_norm"], pos, rot)
            for h in range(HK):
                o = HQ * per + h * HD
                kv[at:at + L, 0, h] = _held64(_prep64(r[:, o:o + HD], s["k_norm"], pos, rot))
                kv[at:at + L, 1, h] = _held64(r[:, o + HK * HD:o + HK * HD + HD])
        if kind != "append":
            for h in range(HK):
                K, V = (_read64(s, b, P + L, h, w) for w in (0, 1))
                if kind == "step":
                    K[P:], V[P:] = kv[at:at + L, 0, h], kv[at:at + L, 1, h]
                Kt = K.T.contiguous()
                for j in range(h * (HQ // HK), (h + 1) * (HQ // HK)):
                    w = q[at:at + L, j] @ Kt / math.sqrt(HD)
                    w = w.masked_fill(torch.arange(P + L, device=DEV)[None] > pos[:, None], float("-inf"))
                    o = torch.softmax(w, 1) @ V
                    if case["gated"]:
                        o = o * torch.sigmoid(r[:, j * per + HD:j * per + 2 * HD])
                    out[at:at + L, j] = o
        at += L
    return {"append": {"q": q, "kv": kv}, "attend": {"out": out}, "step": {"q": q, "kv": kv, "out": out}}[kind]
