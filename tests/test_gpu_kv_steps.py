"""The paged 4-bit K/V cache as a program uses it: prompts, then single tokens, appended and attended layer by layer; calls on a
stream of their own, and captured into a HIP graph and replayed with other batches. Tolerances: tests/test_gpu_kv.py."""
import numpy as np
import pytest

import hybrid_attention as ha
import kv_ref as kr
from test_gpu_kv import DEV, check

pytestmark = pytest.mark.gpu


class Server:
    """Sequences of different lengths on one pool of pages, two layers, and the same in numpy."""

    def __init__(self, prompts, page=16, HQ=8, HK=2, HD=256, rot=64, n_pages=64, seed=0, max_len=512):
        import torch
        self.t, self.rng = torch, np.random.default_rng(seed)
        self.HQ, self.HK, self.HD, self.rot, self.page, self.layers = HQ, HK, HD, rot, page, 2
        self.width = HQ * 2 * HD + 2 * HK * HD
        nb = ha.PagedKV.page_bytes(page, HK, HD)
        self.dpool = torch.full((2, n_pages, nb), 0xFF, dtype=torch.uint8, device=DEV)
        self.kv = ha.PagedKV(self.dpool, n_pages, page_size=page, n_layers=2, max_ctx=max_len, HQ=HQ, HK=HK, HD=HD, rot_dim=rot)
        self.pools = [kr.Pool(n_pages, page, HK, HD, np.full((n_pages, HK, 2, nb // HK // 2), 0xFF, np.uint8)) for _ in range(2)]
        self.w = [[(1 + 0.1 * self.rng.standard_normal(HD)).astype(np.float32) for _ in "qk"] for _ in range(2)]
        for i in range(2):
            self.kv.set_param(i, "q_norm", self.w[i][0])
            self.kv.set_param(i, "k_norm", self.w[i][1])
        self.free = list(self.rng.permutation(n_pages))
        self.tables, self.lens = [[] for _ in prompts], [0] * len(prompts)
        self.stride = self.width + 8
        self.max_len = max_len

    def batch(self, new):
        """Takes pages for new[b] tokens of sequence b; the arrays of a call."""
        for b, n in enumerate(new):
            self.lens[b] += n
            while len(self.tables[b]) * self.page < self.lens[b]:
                self.tables[b].append(self.free.pop())
        stride = self.max_len // self.page
        table = np.full((len(new), stride), -1, np.int32)
        for b, t in enumerate(self.tables):
            table[b, :len(t)] = t
        return np.concatenate([[0], np.cumsum(new)]).astype(np.int32), np.array(self.lens, np.int32), table

    def rows(self, n):
        return self.rng.standard_normal((n, self.stride)).astype(np.float16)

    def expect(self, layer, start, lens, table, rows):
        """Appends in numpy; (queries, outputs) as in 64 bits, the queries rounded as the call's are."""
        HQ, HK, HD = self.HQ, self.HK, self.HD
        pool, (qw, kw) = self.pools[layer], self.w[layer]
        q = np.zeros((len(rows), HQ, HD), np.float16)
        for b in range(len(lens)):
            r = np.arange(start[b], start[b + 1])
            pos = lens[b] - len(r) + np.arange(len(r))
            x = rows[r].astype(np.float64)
            for h in range(HQ):
                q[r, h] = kr.prep(x[:, h * 2 * HD:h * 2 * HD + HD], qw, pos, self.rot).astype(np.float32).astype(np.float16)
            for h in range(HK):
                k0 = HQ * 2 * HD + h * HD
                pool.put_rows(table[b, pos // self.page], pos % self.page, h, 0, kr.prep(x[:, k0:k0 + HD], kw, pos, self.rot).astype(np.float32))
                pool.put_rows(table[b, pos // self.page], pos % self.page, h, 1, x[:, k0 + HK * HD:k0 + HK * HD + HD])
        gate = rows[:, :HQ * 2 * HD].reshape(-1, HQ, 2, HD)[:, :, 1]
        return kr.attend(pool, table, lens, start, q, gate, HQ)


def test_prompts_then_single_tokens():
    s = Server([None] * 5)
    t = s.t
    steps = [[37, 1, 0, 90, 16], [0, 0, 64, 0, 0]] + [[1] * 5] * 4 + [[1, 3, 1, 1, 5], [0, 1, 1, 0, 1]]
    for new in steps:
        start, lens, table = s.batch(new)
        n = sum(new)
        b = ha.KVBatch(5, n, max(new), int(lens.max()), *(t.from_numpy(x).to(DEV) for x in (start, lens, table)), table.shape[1])
        for layer in range(2):
            rows = s.rows(n)
            d = t.from_numpy(rows).to(DEV)
            q = t.empty(n, s.HQ, s.HD, dtype=t.float16, device=DEV)
            out = t.empty_like(q)
            s.kv.append(layer, b, d, s.stride, q)
            s.kv.attention(layer, b, q, d, s.stride, out)
            t.cuda.synchronize()
            want = s.expect(layer, start, lens, table, rows)
            np.testing.assert_array_equal(s.dpool[layer].cpu().numpy().reshape(s.pools[layer].data.shape), s.pools[layer].data)
            check(out.cpu().numpy(), want)


def test_pages_shared_by_two_sequences():
    """A prefix's full pages in two tables: both see them, each appends to pages of its own."""
    s = Server([None] * 2)
    t = s.t
    start, lens, table = s.batch([32, 0])
    s.tables[1] = list(s.tables[0])
    s.lens[1] = 32
    rows = s.rows(32)
    for (st, ln, tb, r) in [(start, lens, table, rows)] + [s.batch([5, 9]) + (s.rows(14),)]:
        d = t.from_numpy(r).to(DEV)
        b = ha.KVBatch(2, len(r), int(np.diff(st).max()), int(ln.max()), *(t.from_numpy(x).to(DEV) for x in (st, ln, tb)), tb.shape[1])
        q = t.empty(len(r), s.HQ, s.HD, dtype=t.float16, device=DEV)
        out = t.empty_like(q)
        s.kv.append(0, b, d, s.stride, q)
        s.kv.attention(0, b, q, d, s.stride, out)
        t.cuda.synchronize()
        check(out.cpu().numpy(), s.expect(0, st, ln, tb, r))


@pytest.mark.parametrize("new,prompt", [([1] * 6, [300, 17, 1, 150, 0, 460]), ([3, 1, 60, 1, 2, 0], [200, 30, 5, 490, 16, 8])])
def test_replays_equal_eager_calls(new, prompt):
    """A captured step, replayed with other rows, lengths and tables, between eager calls on the same handle."""
    s = Server([None] * 6, n_pages=160)
    t = s.t
    st = t.cuda.Stream()
    start, lens, table = s.batch(prompt)
    n = sum(prompt)
    up = lambda x: t.from_numpy(np.ascontiguousarray(x)).to(DEV)  # noqa: E731
    b = ha.KVBatch(6, n, max(prompt), int(lens.max()), up(start), up(lens), up(table), table.shape[1])
    d = up(s.rows(n))
    t.cuda.synchronize()
    for layer in range(2):
        s.kv.append(layer, b, d, s.stride, stream=st.cuda_stream)
    st.synchronize()
    n = sum(new)
    steps = []
    for _ in range(3):
        steps.append([up(x) for x in s.batch(new)] + [up(s.rows(n))])
    live = [x.clone() for x in steps[0]]
    rows = live[3]
    q = t.empty(n, s.HQ, s.HD, dtype=t.float16, device=DEV)
    out, values = t.empty_like(q), t.empty(n, 2, s.HK, s.HD, dtype=t.float16, device=DEV)
    lb = ha.KVBatch(6, n, max(new), s.max_len, *live[:3], table.shape[1])

    def call():
        for layer in range(2):
            s.kv.append(layer, lb, rows, s.stride, q, values, stream=st.cuda_stream)
            s.kv.attention(layer, lb, q, rows, s.stride, out, stream=st.cuda_stream)

    def load(i):
        for a, x in zip(live, steps[i]):
            a.copy_(x)
        for x in (q, out, values):
            x.fill_(float("nan"))

    want = []
    with t.cuda.stream(st):
        for i in range(3):
            load(i)
            call()
            st.synchronize()
            want.append([x.clone() for x in (q, out, values, s.dpool)])
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g, stream=st):
            call()
        for k, i in enumerate([0, 1, 1, 2, 0, 2]):
            if k % 2:
                load((i + 1) % 3)
                call()
                st.synchronize()
            load(i)
            g.replay()
            st.synchronize()
            for x, w in zip((q, out, values), want[i]):
                assert t.equal(x, w), "replay %d" % k
    assert t.equal(s.dpool, want[2][3])


def test_two_handles_on_two_streams():
    """Handles have workspaces of their own: their calls may overlap."""
    import torch as t
    from test_gpu_kv import Call
    a, b = (Call([(2500, 1), (1900, 2)], seed=k) for k in (1, 2))
    wa, wb = a.attention(), b.attention()
    s1, s2 = t.cuda.Stream(), t.cuda.Stream()
    oa, ob = t.empty_like(a.dq), t.empty_like(b.dq)
    t.cuda.synchronize()
    for _ in range(20):
        a.kv.attention(0, a.batch, a.dq, a.drows, a.stride, oa, stream=s1.cuda_stream)
        b.kv.attention(0, b.batch, b.dq, b.drows, b.stride, ob, stream=s2.cuda_stream)
    t.cuda.synchronize()
    np.testing.assert_array_equal(oa.cpu().numpy(), wa)
    np.testing.assert_array_equal(ob.cpu().numpy(), wb)


# every way of sharing out the work (csrc/kv_attn.hip): in a list, planned, in a grid, both kernels, joined and merged
@pytest.mark.parametrize("seqs,heads,page", [
    ([(700, 1), (30, 40), (0, 0)], (8, 2, 256, 64), 16), ([(2000, 20)], (8, 2, 256, 64), 64), ([(0, 3200)], (16, 1, 256, 64), 16),
    ([(40, 1), (0, 1700), (0, 1650), (9, 3)], (16, 1, 256, 64), 32), ([(3, 1)] * 140, (16, 2, 128, 128), 16),
    ([(30, 1)] * 139 + [(3000, 2)], (16, 2, 128, 128), 16)])
def test_captured_calls(seqs, heads, page):
    """Other lengths in the same arrays between replays: a sequence becomes shorter, and long again."""
    import torch as t
    from test_gpu_kv import Call
    c = Call(seqs, heads, page, seed=21)
    st = t.cuda.Stream()
    q, out = t.zeros_like(c.dq), t.zeros_like(c.dq)
    at = max(range(len(seqs)), key=lambda b: seqs[b][0])
    full = int(c.lens[at])
    short = max(full // 2, seqs[at][1])

    def call():
        c.kv.append(0, c.batch, c.drows, c.stride, q, stream=st.cuda_stream)
        c.kv.attention(0, c.batch, q, c.drows, c.stride, out, stream=st.cuda_stream)

    want = {}
    with t.cuda.stream(st):
        for n in (short, full):
            c.dev[1][at] = n
            call()
            st.synchronize()
            want[n] = out.clone(), q.clone(), c.dpool.clone()
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g, stream=st):
            call()
        for k, n in enumerate([full, short, full, full, short, full]):
            if k in (1, 4):
                call()
            c.dev[1][at] = n
            c.dpool.copy_(want[n][2])
            for x in (q, out):
                x.fill_(float("nan"))
            g.replay()
            st.synchronize()
            for x, w in zip((out, q, c.dpool), want[n]):
                assert t.equal(x, w), "replay %d" % k


@pytest.mark.parametrize("new", [[40, 1, 0, 17], [1, 1, 1, 1]])
def test_projections_around_the_cache(new):
    """A layer's attention as a host runs it: hidden rows -> qkv projection -> append -> attention -> output projection, eagerly and
    from a captured graph. Each step is checked against 64 bits on what the one before it left."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "oracle"))
    import mnb_oracle as mo
    s = Server([None] * 4, seed=5)
    t, K, n = s.t, 512, sum(new)
    N1, N2 = s.width, s.HQ * s.HD
    s.stride = N1
    up = lambda x: t.from_numpy(np.ascontiguousarray(x)).to(DEV)  # noqa: E731
    weights = []
    for N, k, size in ((N1, K, 0.01), (K, N2, 0.002)):
        words = s.rng.integers(0, 2 ** 32, (N, k // 32, 4), dtype=np.uint64).astype(np.uint32)
        sc = (size * (0.5 + s.rng.random((N, k // 32)))).astype(np.float16)
        weights.append((ha.MnbWeight(N, k, up(words.view(np.int32)), up(sc)), mo.dequant(words, sc, N, k)))
    (w1, W1), (w2, W2) = weights
    start, lens, table = s.batch([30, 200, 5, 0])  # a prompt, so that the cache is not empty
    rows = s.rows(235)
    b0 = ha.KVBatch(4, 235, 200, 200, up(start), up(lens), up(table), table.shape[1])
    s.kv.append(0, b0, up(rows), N1)
    s.expect(0, start, lens, table, rows)
    start, lens, table = s.batch(new)
    x = s.rng.standard_normal((n, K)).astype(np.float16)
    d, big = up(x), t.empty(n, N1, dtype=t.float16, device=DEV)
    b = ha.KVBatch(4, n, max(new), int(lens.max()), up(start), up(lens), up(table), table.shape[1])
    q, mix, y = (t.empty(n, *k, dtype=t.float16, device=DEV) for k in ((s.HQ, s.HD), (s.HQ, s.HD), (K,)))
    st = t.cuda.Stream()
    t.cuda.synchronize()

    def layer():
        w1.forward_noalloc(n, d, big, stream=st.cuda_stream)
        s.kv.append(0, b, big, N1, q, stream=st.cuda_stream)
        s.kv.attention(0, b, q, big, N1, mix, stream=st.cuda_stream)
        w2.forward_noalloc(n, mix, y, stream=st.cuda_stream)

    layer()
    st.synchronize()
    big_h, mix_h = big.cpu().numpy(), mix.cpu().numpy()
    # projections: f16 weights (a code times a scale, rounded) and outputs, f32 sums: 2^-11 each of the largest element at most
    assert mo.rel_err(big_h.astype(np.float64), mo.matmul(x, W1)) <= 2 ** -10
    check(mix_h, s.expect(0, start, lens, table, big_h))
    np.testing.assert_array_equal(s.dpool[0].cpu().numpy().reshape(s.pools[0].data.shape), s.pools[0].data)
    assert mo.rel_err(y.cpu().numpy().astype(np.float64), mo.matmul(mix_h.reshape(n, N2), W2)) <= 2 ** -10
    want = y.clone()
    g = t.cuda.CUDAGraph()
    with t.cuda.stream(st):
        with t.cuda.graph(g, stream=st):
            layer()
        for k in range(3):
            if k == 1:
                layer()
            for z in (big, q, mix, y):
                z.fill_(float("nan"))
            g.replay()
            st.synchronize()
            assert t.equal(y, want), "replay %d" % k
