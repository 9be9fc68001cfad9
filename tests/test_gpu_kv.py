"""The paged 4-bit K/V cache (ha_kv_append, ha_kv_attention) against numpy in 64 bits (tests/kv_ref.py).

Tolerances. q: f32 arithmetic, one rounding to f16 (2^-11 of the value) and what a few hundred f32 roundings of the norm and the
rotation leave (2^-24 each, of the row's largest value): 2^-11 |q| + 2^-15. Codes, scales and zeros: equal. values: the f16
rounding of what the codes stand for: equal. Attention: f16 operands (the dequantised rows or the weighted probabilities: 2^-11
each) with f32 sums and an f16 output: each output is a weighted mean of the values v_j, so an error of 2^-11 in p_j and in v_j
each moves it by at most 2^-10 max|v|, one of the scores, |q||k| 2^-11 scale at the most, by as much of max|v| again: with |scale
q.k| <= 8 in these inputs 2^-8 max|v|, a bound that random roundings do not come near; the norm of the error is held to 2^-10 of
the norm of the output, three times the rounding of the output and of P and the rows (2^-11 / sqrt(3) each) together."""
import numpy as np
import pytest

import hybrid_attention as ha
import kv_ref as kr

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HEADS = [(8, 2, 256, 64), (16, 2, 128, 128), (4, 4, 128, 64), (3, 1, 256, 0), (16, 1, 128, 8), (7, 1, 256, 256)]


class Call:
    """A cache with random pages, and a ragged batch on it."""

    def __init__(self, seqs, heads=HEADS[0], page=16, gated=True, f32=False, seed=0, extra=0, max_ctx=None, garbage=True, **kw):
        import torch
        self.torch = torch
        rng = self.rng = np.random.default_rng(seed)
        self.HQ, self.HK, self.HD, self.rot = heads
        self.gated, self.seqs, self.page = gated, seqs, page
        self.lens = np.array([p + n for p, n in seqs], np.int32)
        self.start = np.concatenate([[0], np.cumsum([n for _, n in seqs])]).astype(np.int32)
        need = [-(-int(n) // page) for n in self.lens]
        self.width = max(need + [1]) + 1
        self.n_pages = sum(need) + 2
        self.table = np.full((len(seqs), self.width), -1, np.int32)
        ids, at = rng.permutation(self.n_pages), 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        # slots that hold no token: every byte pattern, NaN and infinite scales among them
        blk = page * (self.HD // 2 + 16)
        fill = rng.integers(0, 256, (self.n_pages, self.HK, 2, blk), dtype=np.uint8) if garbage else np.zeros((self.n_pages, self.HK, 2, blk), np.uint8)
        if garbage:
            fill[..., page * self.HD // 2:] = np.where(rng.random((self.n_pages, self.HK, 2, page * 16)) < 0.5, 0xFF, fill[..., page * self.HD // 2:])
        self.pool = kr.Pool(self.n_pages, page, self.HK, self.HD, fill)
        for b in range(len(seqs)):
            t = np.arange(self.lens[b])
            for h in range(self.HK):
                for w in (0, 1):
                    self.pool.put_rows(self.table[b, t // page], t % page, h, w, rng.standard_normal((len(t), self.HD)))
        self.T = int(self.start[-1])
        self.n_rows = self.T + extra
        self.max_rows = max([n for _, n in seqs] + [0])
        self.max_len = int(max(list(self.lens) + [1]))
        self.stride = self.HQ * self.HD * (2 if gated else 1) + 2 * self.HK * self.HD + (0 if gated else 8)  # (some rows with padding)
        self.rows = rng.standard_normal((max(self.n_rows, 1), self.stride)).astype(np.float32 if f32 else np.float16)
        self.qw, self.kw = ((1 + 0.1 * rng.standard_normal(self.HD)).astype(np.float32) for _ in "qk")
        self.dpool = torch.from_numpy(self.pool.data.copy()).to(DEV)
        self.kv = ha.PagedKV(self.dpool, self.n_pages, page_size=page, max_ctx=max_ctx or self.max_len, HQ=self.HQ, HK=self.HK, HD=self.HD,
                             rot_dim=self.rot, gated=gated, dtype=ha.F32 if f32 else ha.F16, **kw)
        self.kv.set_param(0, "q_norm", self.qw)
        self.kv.set_param(0, "k_norm", self.kw)
        self.drows = torch.from_numpy(self.rows).to(DEV)
        self.dev = [torch.from_numpy(a).to(DEV) for a in (self.start, self.lens, self.table)]
        self.batch = self.make_batch()
        self.q = rng.standard_normal((max(self.n_rows, 1), self.HQ, self.HD)).astype(np.float16)
        self.dq = torch.from_numpy(self.q).to(DEV)

    def make_batch(self, **kw):
        d = dict(n_seqs=len(self.seqs), n_rows=self.n_rows, max_rows=self.max_rows, max_len=self.max_len, row_start=self.dev[0],
                 lens=self.dev[1], pages=self.dev[2], table_stride=self.width)
        if "n_seqs" in kw:  # (as plain addresses: KVBatch refuses tensors that end too early, the library the number)
            d.update({k: d[k].data_ptr() for k in ("row_start", "lens", "pages")})
        d.update(kw)
        return ha.KVBatch(**d)

    def gates(self):
        if not self.gated:
            return None
        return self.rows[:, :self.HQ * 2 * self.HD].reshape(-1, self.HQ, 2, self.HD)[:, :, 1]

    def append(self, batch=None, **kw):
        t = self.torch
        q = t.full((max(self.n_rows, 1), self.HQ, self.HD), 7.0, dtype=t.float16, device=DEV)
        v = t.full((max(self.n_rows, 1), 2, self.HK, self.HD), 7.0, dtype=t.float16, device=DEV)
        self.kv.append(0, batch or self.batch, self.drows, self.stride, q, v, **kw)
        t.cuda.synchronize()
        return q.cpu().numpy(), v.cpu().numpy(), self.dpool.cpu().numpy()

    def attention(self, batch=None, q=None, **kw):
        t = self.torch
        out = t.full((max(self.n_rows, 1), self.HQ, self.HD), 7.0, dtype=t.float16, device=DEV)
        self.kv.attention(0, batch or self.batch, self.dq if q is None else q, self.drows if self.gated else None, self.stride if self.gated else 0, out, **kw)
        t.cuda.synchronize()
        return out.cpu().numpy()

    def expected(self, rows=None, q=None):
        return kr.attend(self.pool, self.table, self.lens, self.start, self.q if q is None else q, self.gates(), self.HQ, rows=rows)


def check(got, want, vmax=4.5):
    """got [n_rows][HQ][HD] against want {row: [HQ][HD]}."""
    e = np.stack([got[t].astype(np.float64) - want[t] for t in sorted(want)])
    w = np.stack([want[t] for t in sorted(want)])
    assert np.isfinite(e).all()
    rel, big = np.linalg.norm(e) / np.linalg.norm(w), np.abs(e).max()
    print("rel %.2e max %.2e" % (rel, big))
    assert rel <= 2 ** -10 and big <= vmax * 2 ** -8


# ---- append ----

def check_append(c, q, v, pool):
    per = c.HD * (2 if c.gated else 1)
    n_q = c.HQ * per
    for b in range(len(c.seqs)):
        r = np.arange(c.start[b], c.start[b + 1])
        pos = c.lens[b] - len(r) + np.arange(len(r))
        x = c.rows[r].astype(np.float64)
        for h in range(c.HQ):
            want = kr.prep(x[:, h * per:h * per + c.HD], c.qw, pos, c.rot)
            assert (np.abs(q[r, h] - want) <= 2 ** -11 * np.abs(want) + 2 ** -15).all()
        for h in range(c.HK):
            k = kr.prep(x[:, n_q + h * c.HD:n_q + (h + 1) * c.HD], c.kw, pos, c.rot).astype(np.float32)
            vv = x[:, n_q + (c.HK + h) * c.HD:n_q + (c.HK + h + 1) * c.HD].astype(np.float32)
            for w, rows in ((0, k), (1, vv)):
                c.pool.put_rows(c.table[b, pos // c.page], pos % c.page, h, w, rows)
                held = kr.values(*kr.quantise(rows))
                with np.errstate(all="ignore"):
                    np.testing.assert_array_equal(v[r, w, h], held.astype(np.float32).astype(np.float16))
    np.testing.assert_array_equal(pool, c.pool.data)  # the new rows, and every other byte as it was
    assert (q[c.T:] == 7).all() and (v[c.T:] == 7).all()


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("gated,f32,page", [(True, False, 16), (False, True, 32), (True, True, 64), (False, False, 128)])
def test_append(heads, gated, f32, page):
    c = Call([(0, 1), (15, 1), (0, 37), (5, 0), (30, 5), (63, 66)], heads, page, gated, f32, seed=1, extra=2)
    check_append(c, *c.append())


def test_append_far_positions():
    c = Call([(0, 3), (0, 2)], page=256, seed=2)
    far = np.array([131072, 100001], np.int32)  # positions of a long context; its other pages are not touched
    c.kv = ha.PagedKV(c.dpool, c.n_pages, page_size=256, max_ctx=131072)
    c.kv.set_param(0, "q_norm", c.qw)
    c.kv.set_param(0, "k_norm", c.kw)
    c.lens, c.width = far, 512
    table = np.full((2, 512), -1, np.int32)
    table[0, 511], table[1, 390] = 0, 1
    c.table = table
    c.dev = [c.torch.from_numpy(a).to(DEV) for a in (c.start, c.lens, c.table)]
    c.max_len = 131072
    c.batch = c.make_batch()
    check_append(c, *c.append())


def test_append_values_that_do_not_fit():
    """All values equal, huge, infinite or NaN in one group: the group alone is zero-scaled or NaN."""
    c = Call([(3, 8)], HEADS[1], 16, True, True, seed=3)
    HD, n_q = c.HD, c.HQ * 2 * c.HD
    v = c.rows[:, n_q + c.HK * HD:]
    v[0, :32] = 1.5
    v[1, 5], v[2, 40], v[3, 70] = np.nan, np.inf, -np.inf
    v[4, :32], v[5, :16] = 3e38, 60000.0
    v[5, 16:32] = -65000.0
    v[6, :HD] = 0
    v[7, :32] = np.linspace(1e-7, 2e-7, 32)
    c.drows = c.torch.from_numpy(c.rows).to(DEV)
    check_append(c, *c.append())
    got = c.dpool.cpu().numpy()
    p = kr.Pool(c.n_pages, c.page, c.HK, HD, got).read(c.table[0][np.arange(3, 11) // 16], np.arange(3, 11) % 16, 0, 1)
    assert (p[0, :32] == 1.5).all() and (p[6] == 0).all()
    for row, group in ((1, 0), (2, 1), (3, 2), (4, 0)):
        assert np.isnan(p[row, 32 * group:32 * group + 32]).all() and np.isnan(p[row]).sum() == 32


def test_append_without_outputs():
    c = Call([(10, 9)], seed=4)
    want = c.append()[2].copy()
    c.dpool.copy_(c.torch.from_numpy(c.pool.data))
    c.kv.append(0, c.batch, c.drows, c.stride)
    c.torch.cuda.synchronize()
    np.testing.assert_array_equal(c.dpool.cpu().numpy(), want)


# ---- attention ----

@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("gated,f32,page", [(True, False, 16), (False, False, 64), (True, True, 32)])
def test_attention_ragged(heads, gated, f32, page):
    c = Call([(0, 1), (15, 1), (0, 37), (5, 0), (130, 5), (63, 66), (200, 1)], heads, page, gated, f32, seed=5, extra=3)
    got = c.attention()
    check(got[:c.T], c.expected())
    assert (got[c.T:] == 7).all()


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257])
@pytest.mark.parametrize("heads", HEADS[:2])
def test_attention_one_token(n, heads):
    c = Call([(n - 1, 1)], heads, 16, seed=n)
    check(c.attention(), c.expected())


@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 64, 65, 100, 129, 260])
@pytest.mark.parametrize("heads,P", [(HEADS[0], 0), (HEADS[0], 77), (HEADS[1], 50), (HEADS[2], 0), (HEADS[3], 13)])
def test_attention_row_counts(n, heads, P):
    c = Call([(P, n)], heads, 32, seed=n)
    check(c.attention(), c.expected())


def test_attention_many_sequences():
    rng = np.random.default_rng(6)
    c = Call([(int(p), 1) for p in rng.integers(0, 90, 70)], page=16, seed=6)
    check(c.attention(), c.expected())


@pytest.mark.parametrize("B,P,n,heads", [(1, 3000, 1, HEADS[0]), (3, 1700, 1, HEADS[0]), (1, 2100, 61, HEADS[0]), (2, 900, 300, HEADS[1])])
def test_attention_long(B, P, n, heads):
    c = Call([(P, n)] * B, heads, 64, seed=7)
    rows = set(range(0, c.T, max(1, c.T // 24))) | {c.T - 1}
    want = c.expected(rows=rows)
    check(c.attention(), want)


def test_attention_peaked_and_extreme_scores():
    """Scores up to several hundred: one key takes all, running maxima rise by more than f16 spans."""
    c = Call([(300, 3), (40, 1)], page=16, seed=8)
    c.q[:] = c.q * np.float16(40)
    c.dq = c.torch.from_numpy(c.q).to(DEV)
    got, want = c.attention(), c.expected()
    e = max(np.abs(got[t] - want[t]).max() for t in want)
    # a score's error, f32 sums of 256 terms and f16 rows, is 2^-11 |score| at the most: with scores up to 400 a factor
    # exp(0.2) between two keys' weights
    assert np.isfinite(got).all() and e <= 0.25 * 4.5


def test_attention_masked_infinities():
    """A NaN token (a group that reads as NaN) reaches the rows that see it and no other."""
    c = Call([(40, 6)], HEADS[0], 16, seed=9)
    row = c.rng.standard_normal(c.HD)
    row[3] = np.inf
    c.pool.put(c.table[0, 44 // 16], 44 % 16, 0, 1, row)
    c.pool.put(c.table[0, 45 // 16], 45 % 16, 1, 0, row)
    c.dpool.copy_(c.torch.from_numpy(c.pool.data))
    got = c.attention()
    want = c.expected(rows={0, 1, 2, 3})
    check(got, want)
    assert np.isnan(got[4:, :4, :64]).all() and np.isfinite(got[4:, :4, 64:]).all()
    assert np.isnan(got[5, 4:]).all() and np.isfinite(got[4, 4:]).all()


def test_attention_scale():
    c = Call([(50, 2)], page=16, seed=10, scale=0.11)
    check(c.attention(), kr.attend(c.pool, c.table, c.lens, c.start, c.q, c.gates(), c.HQ, scale=np.float32(0.11)))


# ---- what does not fit ----

def test_bad_pages():
    c = Call([(70, 3), (20, 2), (33, 1)], page=16, seed=11)
    c.table[0, 4] = c.n_pages  # tokens 64 .. 72: rows 0 .. 2 see them
    c.table[1, 0] = -5
    c.dev[2].copy_(c.torch.from_numpy(c.table))
    got = c.attention()
    assert np.isnan(got[:5]).all()
    c2 = {t: w for t, w in kr.attend(c.pool, c.table % c.n_pages, c.lens, c.start, c.q, c.gates(), c.HQ, rows={5}).items()}
    check(got, c2)
    before = c.dpool.cpu().numpy()
    q, v, pool = c.append()
    assert np.isfinite(q).all() and np.isnan(v[:3]).all() and np.isfinite(v[3:]).all()
    same = (pool == before).all(axis=(1, 2, 3))
    touched = {int(c.table[1, 1]), int(c.table[2, 2])}
    assert set(np.nonzero(~same)[0]) == touched


@pytest.mark.parametrize("what", ["len over max_len", "more rows than max_rows", "fewer tokens than rows", "row_start falls", "row_start past the rows", "negative"])
def test_sequences_that_do_not_fit(what):
    c = Call([(20, 2), (30, 3), (40, 2)], page=16, seed=12, max_ctx=64)
    start, lens = c.start.copy(), c.lens.copy()
    nan = {2, 3, 4}
    if what == "len over max_len":
        lens[1] = c.max_len + 1
    elif what == "more rows than max_rows":
        c.batch = c.make_batch(max_rows=2)
        nan = {2, 3}
    elif what == "fewer tokens than rows":
        lens[1] = 2
    elif what == "row_start falls":
        start[1], start[2] = 5, 2  # the first sequence takes rows 0 .. 4 (more than max_rows), the last 2 .. 6
        nan = {0, 1, 2}
    elif what == "row_start past the rows":
        start[3], nan = 1000, {5, 6}
    else:
        start[0], nan = -1, {0, 1}
    c.dev[0].copy_(c.torch.from_numpy(start))
    c.dev[1].copy_(c.torch.from_numpy(lens))
    before = c.dpool.cpu().numpy()
    got = c.attention()
    q, v, pool = c.append()
    if what == "row_start falls":  # rows of two sequences: written by both
        assert np.isnan(got[:2]).all() and np.isnan(q[:2]).all() and np.isnan(v[:2]).all()
        return
    for t in range(c.T):
        for x in (got, q, v):
            assert np.isnan(x[t]).all() if t in nan else np.isfinite(x[t]).all() or (x[t] == 7).all()
    fine = [b for b in range(3) if start[b] not in nan and (b, what) != (0, "negative") and (b, what) != (2, "row_start past the rows") and
            not (b == 1 and what not in ("row_start past the rows", "negative"))]
    want = {t: w for t, w in c.expected().items() if any(c.start[b] <= t < c.start[b + 1] for b in fine)}
    check(got, want)
    changed = set(np.nonzero((pool != before).any(axis=(1, 2, 3)))[0])
    assert changed == {int(c.table[b, p // 16]) for b in fine for p in range(c.lens[b] - (c.start[b + 1] - c.start[b]), c.lens[b])}


def test_refusals():
    c = Call([(20, 2)], page=16, seed=13, max_ctx=64)
    out = c.dq.clone()

    def refused(code, f, *a, **k):
        with pytest.raises(ha.HAError) as ei:
            f(*a, **k)
        assert ei.value.code == code

    for kw, code in [(dict(max_len=65), ha.HA_ERR_CONTEXT), (dict(max_len=49), ha.HA_ERR_ARG), (dict(n_seqs=0), ha.HA_ERR_ARG),
                     (dict(n_seqs=65536), ha.HA_ERR_ARG), (dict(max_rows=3), ha.HA_ERR_ARG), (dict(n_rows=-1), ha.HA_ERR_ARG),
                     (dict(max_len=1), ha.HA_ERR_ARG), (dict(row_start=None), ha.HA_ERR_ARG), (dict(lens=None), ha.HA_ERR_ARG),
                     (dict(pages=None), ha.HA_ERR_ARG), (dict(table_stride=0), ha.HA_ERR_ARG)]:
        b = c.make_batch(**kw)
        refused(code, c.kv.append, 0, b, c.drows, c.stride)
        refused(code, c.kv.attention, 0, b, c.dq, c.drows, c.stride, out)
    p = c.drows.data_ptr()
    for layer in (-1, 1):
        refused(ha.HA_ERR_ARG, c.kv.append, layer, c.batch, c.drows, c.stride)
        refused(ha.HA_ERR_ARG, c.kv.attention, layer, c.batch, c.dq, c.drows, c.stride, out)
        refused(ha.HA_ERR_ARG, c.kv.set_param, layer, "q_norm", c.qw)
    for rows, stride in ((None, c.stride), (p + 2, c.stride), (c.drows, c.stride - 8), (c.drows, c.stride + 4)):
        refused(ha.HA_ERR_ARG, c.kv.append, 0, c.batch, rows, stride)
        refused(ha.HA_ERR_ARG, c.kv.attention, 0, c.batch, c.dq, rows, stride, out)
    refused(ha.HA_ERR_ARG, c.kv.append, 0, c.batch, c.drows, c.stride, out.data_ptr() + 2)
    refused(ha.HA_ERR_ARG, c.kv.append, 0, c.batch, c.drows, c.stride, out, out.data_ptr() + 8)
    for q, o in ((None, out), (c.dq, None), (c.dq.data_ptr() + 8, out), (c.dq, out.data_ptr() + 8)):
        refused(ha.HA_ERR_ARG, c.kv.attention, 0, c.batch, q, c.drows, c.stride, o)
    refused(ha.HA_ERR_PARAM, c.kv.set_param, 0, "conv", c.qw)
    refused(ha.HA_ERR_PARAM, c.kv.set_param, 0, "q_norm", c.qw[:-1])
    with pytest.raises(ha.HAError) as ei:
        ha.PagedKV(c.dpool, 4, device=99)
    assert ei.value.code == ha.HA_ERR_ARG


def test_calls_without_rows():
    c = Call([(20, 0), (3, 0)], page=16, seed=14)
    q, v, pool = c.append()
    assert (q == 7).all() and (v == 7).all()
    np.testing.assert_array_equal(pool, c.pool.data)
    assert (c.attention() == 7).all()
