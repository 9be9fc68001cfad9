"""ha_kv_attention and ha_kv_append on batches whose work is shared out in other ways (csrc/kv_attn.hip, "who does what"): many rows a
sequence, equal and ragged, beside single tokens; more sequences than one wave has lanes, and more than are listed; long pieces.
Tolerances: tests/test_gpu_kv.py."""
import numpy as np
import pytest

import hybrid_attention as ha
import kv_ref as kr
from test_gpu_kv import Call, check, check_append

pytestmark = pytest.mark.gpu
H16 = (16, 1, 256, 64)   # 16 query heads on one KV head: 8 rows are a block of 128 columns
H8 = (16, 2, 128, 128)
MODEL = (8, 2, 256, 64)


def some(c, n=40, seed=0):
    """Rows to check: the first and last of every sequence, and n others."""
    rng = np.random.default_rng(seed)
    ends = {int(t) for b in range(len(c.seqs)) if c.seqs[b][1] for t in (c.start[b], c.start[b + 1] - 1)}
    if len(ends) > 60:
        ends = set(rng.permutation(sorted(ends))[:60].tolist())
    return ends | set(rng.integers(0, c.T, n).tolist())


# columns x KV heads / 128 is at least 384 in all of these: the kernel of many columns
@pytest.mark.parametrize("seqs,heads,page,gated", [
    ([(0, 800)] * 4, H8, 16, False),                                   # equal
    ([(37, 1600)] * 2, H16, 64, True),                                 # behind a prefix
    ([(0, 3100)], H16, 32, False),                                     # one
    ([(0, 1), (5, 900), (0, 1333), (700, 1), (64, 1000), (3, 0), (31, 17)], H16, 16, True),   # ragged, single tokens among them
    ([(100, 6300)], MODEL, 128, True)])
def test_many_rows(seqs, heads, page, gated):
    c = Call(seqs, heads, page, gated, seed=1, extra=2)
    got = c.attention()
    check(got[:c.T], c.expected(rows=some(c)))
    assert np.isfinite(got[:c.T].astype(np.float32)).all() and (got[c.T:] == 7).all()


def test_many_rows_of_more_than_64_sequences():
    rng = np.random.default_rng(2)
    c = Call([(int(p), int(n)) for p, n in zip(rng.integers(0, 40, 90), rng.integers(0, 90, 90))], H16, 16, seed=2)
    assert c.T * 16 // 128 >= 384
    check(c.attention(), c.expected(rows=some(c)))


@pytest.mark.parametrize("n", [64, 65, 100, 128, 129, 140])
def test_single_tokens_of_many_sequences(n):
    rng = np.random.default_rng(n)
    c = Call([(int(p), 1) for p in rng.integers(0, 300, n)], (3, 1, 256, 0), 16, False, seed=n)
    check(c.attention(), c.expected())


@pytest.mark.parametrize("n,heads", [(30, MODEL), (130, (3, 1, 256, 0)), (200, (4, 4, 128, 64))])
def test_some_long_sequences(n, heads):
    """A few sequences are cut into pieces, the others are shorter than one."""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 60, n)
    lens[[1, n // 2, n - 1]] = [2600, 1500, 2047]
    c = Call([(int(p), 1 + int(i % 5 == 0)) for i, p in enumerate(lens)], heads, 16, seed=n)
    rows = some(c, 20) | {int(c.start[b]) for b in (1, n // 2, n - 1)}
    check(c.attention(), c.expected(rows=rows))


@pytest.mark.parametrize("P,n,heads", [(40000, 1, (16, 1, 128, 8)), (33000, 2, (2, 2, 128, 8)), (9000, 20, MODEL)])
def test_pieces_of_a_long_context(P, n, heads):
    """Pieces longer than 1024 keys (the first two: 40000 x 1 unit over 512 is one step a wave; the same over few units is not)."""
    c = Call([(P, n)], heads, 256, seed=3)
    check(c.attention(), c.expected(rows={0, n - 1}))


def test_long_pieces_of_many_sequences():
    """130 equal sequences in a grid of pieces of 1024 keys and more."""
    c = Call([(2300, 1)] * 130, (4, 4, 128, 8), 256, False, seed=4)
    check(c.attention(), c.expected(rows={0, 64, 129}))


def test_append_many_rows():
    c = Call([(0, 2100), (5, 1500)], (16, 2, 128, 128), 32, False, seed=5, extra=1)
    check_append(c, *c.append())
    c = Call([(0, 700), (33, 1200), (7, 1)], MODEL, 16, True, True, seed=6)
    check_append(c, *c.append())


@pytest.mark.parametrize("heads", [H8, H16])
def test_sequences_that_do_not_fit_among_many_rows(heads):
    c = Call([(0, 1100), (10, 1300), (0, 40), (20, 1), (0, 900)], heads, 16, seed=7)
    start, lens = c.start.copy(), c.lens.copy()
    lens[1] = 900         # fewer tokens than rows
    lens[3] = -4
    c.dev[1].copy_(c.torch.from_numpy(lens))
    got = c.attention()
    bad = np.r_[start[1]:start[2], start[3]:start[4]]
    assert np.isnan(got[bad].astype(np.float32)).all()
    check(got, {t: w for t, w in c.expected(rows=some(c)).items() if t not in set(bad.tolist())})


def test_bad_page_among_many_rows():
    c = Call([(0, 3200)], H16, 16, seed=8)
    c.table[0, 150] = -1  # tokens 2400 .. 2415
    c.dev[2].copy_(c.torch.from_numpy(c.table))
    got = c.attention()
    assert np.isnan(got[2400:].astype(np.float32)).all()
    check(got, kr.attend(c.pool, c.table % c.n_pages, c.lens, c.start, c.q, c.gates(), c.HQ, rows={0, 5, 1000, 2399}))


@pytest.mark.parametrize("seqs,heads", [([(3000, 1)], MODEL), ([(900, 3), (40, 1), (1700, 2)], MODEL), ([(0, 3200)], H16), ([(2000, 60)], MODEL)])
def test_the_same_call_gives_the_same_bits(seqs, heads):
    """Also after a call of another shape, which leaves other results in the workspace."""
    c = Call(seqs, heads, 64, seed=9)
    first = c.attention()
    small = c.make_batch(n_seqs=1, n_rows=min(c.T, 5), max_rows=min(c.T, 5))
    for _ in range(3):
        c.attention(batch=small)
        np.testing.assert_array_equal(c.attention().view(np.uint16), first.view(np.uint16))


# one sequence has most of the rows: append's rows are found in a list (csrc/kv.hip, find_rows)
@pytest.mark.parametrize("seqs,heads", [
    ([(7, 1)] * 5 + [(3, 90), (0, 0), (9, 3)] + [(30, 1)] * 4, MODEL),
    ([(int(p), 1) for p in range(70)] + [(11, 200)] + [(4, 2), (0, 0)] * 10, H8),
    ([(2, 130)] + [(5, 1)] * 150, (3, 1, 256, 0))])
def test_append_of_one_long_sequence(seqs, heads):
    c = Call(seqs, heads, 16, True, seed=10, extra=2)
    check_append(c, *c.append())


def test_append_of_one_long_sequence_that_does_not_fit():
    c = Call([(7, 1)] * 6 + [(3, 90), (9, 3)], MODEL, 16, True, seed=11)
    lens = c.lens.copy()
    lens[[2, 6]] = 0
    c.dev[1].copy_(c.torch.from_numpy(lens))
    before = c.dpool.cpu().numpy()
    q, v, pool = c.append()
    bad = np.zeros(c.T, bool)
    bad[2] = bad[6:96] = True
    for x in (q, v):
        assert np.isnan(x[bad]).all() and np.isfinite(x[~bad]).all()
    changed = set(np.nonzero((pool != before).any(axis=(1, 2, 3)))[0])
    assert changed == {int(c.table[b, p // 16]) for b in (0, 1, 3, 4, 5, 7) for p in range(c.lens[b] - (c.start[b + 1] - c.start[b]), c.lens[b])}


# more than 128 sequences: contexts of up to 1024 keys in a grid, others by a plan of the pieces
@pytest.mark.parametrize("n,heads,long,rows", [
    (129, MODEL, 1100, 1), (300, (3, 1, 256, 0), 5000, 1), (150, H8, 2100, 5), (200, (4, 4, 128, 64), 300, 7), (1500, H8, 1500, 1),
    (5000, (16, 1, 128, 8), 1700, 1), (4500, (16, 1, 128, 8), 20, 1), (140, H16, 3100, 40)])
def test_plans(n, heads, long, rows):
    """Some sequences longer than a piece, some without rows, some that do not fit."""
    rng = np.random.default_rng(n)
    seqs = [(int(p), int(r)) for p, r in zip(rng.integers(0, 30, n), rng.integers(0, 2, n))]
    for at in (0, 3, n // 2, n - 1):
        seqs[at] = (int(long * rng.uniform(0.4, 1.0)), rows)
    c = Call(seqs, heads, 16, heads[2] == 256, seed=n)
    lens = c.lens.copy()
    bad = [b for b in (2, n // 3, n - 2) if seqs[b][1]]
    lens[bad] = -1
    c.dev[1].copy_(c.torch.from_numpy(lens))
    got = c.attention()
    out = np.zeros(c.T, bool)
    for b in bad:
        out[c.start[b]:c.start[b + 1]] = True
    assert np.isnan(got[out]).all() and np.isfinite(got[~out]).all()
    check(got, c.expected(rows={t for t in some(c) if not out[t]}))


# pieces joined in groups (one row of up to 4 columns of 256 channels, 8 of 128), by the last one, and merged
@pytest.mark.parametrize("P,n,heads", [
    (1900, 1, MODEL), (2100, 1, MODEL), (2500, 1, H8), (8200, 1, MODEL), (12000, 1, H8), (33500, 1, MODEL), (40000, 1, (1, 1, 256, 64)),
    (2100, 2, MODEL), (1000, 4, MODEL), (8200, 2, H8), (900, 9, H16)])
def test_joins(P, n, heads):
    """Three times, with a shorter call between: the counts are zero again, what the workspace holds does not matter."""
    c = Call([(P, n)], heads, 64, seed=12)
    first = c.attention()
    check(first, c.expected(rows={0, n - 1}))
    for _ in range(2):
        c.dev[1].fill_(P // 2 + n)
        c.attention()
        c.dev[1].fill_(P + n)
        np.testing.assert_array_equal(c.attention().view(np.uint16), first.view(np.uint16))


@pytest.mark.parametrize("size", [2e-4, 0.05, 300.0, 2e4])
@pytest.mark.parametrize("seqs,heads", [([(900, 3), (40, 1)], MODEL), ([(300, 20)], H8), ([(0, 3200)], H16)])
def test_sizes_of_values(seqs, heads, size):
    """Values from f16's subnormal scales to its largest: P times a scale stays an f16."""
    c = Call(seqs, heads, 16, False, seed=14)
    for b in range(len(seqs)):
        t = np.arange(c.lens[b])
        for h in range(c.HK):
            c.pool.put_rows(c.table[b, t // 16], t % 16, h, 1, np.clip(size * c.rng.standard_normal((len(t), c.HD)), -6e4, 6e4))
    c.dpool.copy_(c.torch.from_numpy(c.pool.data))
    c.q[:] = c.q * np.float16(3)  # (maxima that rise)
    c.dq = c.torch.from_numpy(c.q).to("cuda:0")
    got, want = c.attention(), c.expected(rows=some(c))
    e = np.stack([got[t].astype(np.float64) - want[t] for t in sorted(want)])
    w = np.stack([want[t] for t in sorted(want)])
    # as check(), and f16's steps of 2^-24 in the output and in the products P s, which stand against P of 1 and more and up to 8 codes
    assert np.isfinite(e).all() and np.linalg.norm(e) <= 2 ** -9 * np.linalg.norm(w) + 9 * 2 ** -25 * np.sqrt(e.size)


# (the first sequence's rows, sequences, the last one's length, heads): in a list, planned, of many columns
@pytest.mark.parametrize("rows,n,long,heads", [(64, 59, 1800, MODEL), (40, 201, 2500, MODEL), (3000, 9, 3300, H16)])
def test_row_start_that_falls_again_and_again(rows, n, long, heads):
    """Every second sequence claims the first one's rows: those stay the first one's, the others store nothing, and no work is left
    half done that a later call on the handle would find."""
    c = Call([(0, rows)] + [(rows, 0)] * (n - 2) + [(long, 0)], heads, 16, seed=15, extra=1)
    c.max_len = long
    good = c.dev[0].clone()
    c.dev[0][::2], c.dev[0][1::2] = 0, rows
    c.batch = c.make_batch()
    got = c.attention()
    check(got[:rows], c.expected(rows=set(range(rows)) if rows < 100 else {0, 1, 500, rows - 1}))
    assert (got[rows:] == 7).all()
    check_append(c, *c.append())
    # the last sequence's rows, in pieces, on this handle and on one that has seen no other call
    c.dev[0].copy_(good)
    c.dev[0][:n] = 0
    one = c.make_batch()
    first = c.attention(batch=one)
    c.kv = ha.PagedKV(c.dpool, c.n_pages, page_size=16, max_ctx=long, HQ=c.HQ, HK=c.HK, HD=c.HD, rot_dim=c.rot)
    want = c.attention(batch=one)
    assert np.isfinite(want[:rows]).all()
    np.testing.assert_array_equal(first.view(np.uint16), want.view(np.uint16))


def shared_pages(seqs, heads, n_pages, page=256, seed=0, pool=None, **kw):
    """A call whose sequences take their full pages from one pool, over and over, in an order of their own (contexts of many pages)."""
    c = Call([(n_pages * page - n, n) if b == 0 else (0, n) for b, (_, n) in enumerate(seqs)], heads, page, False, seed=seed, max_ctx=max(p + n for p, n in seqs), **kw)
    ids = c.table[0, :n_pages].copy()
    c.lens = np.array([p + n for p, n in seqs], np.int32)
    assert (c.lens % page == 0).all()
    c.width = int(c.lens.max()) // page
    c.table = np.stack([c.rng.permutation(np.resize(ids, c.width)) for _ in seqs]).astype(np.int32)
    c.max_len = int(c.lens.max())
    c.dev = [c.torch.from_numpy(a).to("cuda:0") for a in (c.start, c.lens, c.table)]
    c.batch = c.make_batch()
    if pool is not None:
        pool(c, ids)
        c.dpool.copy_(c.torch.from_numpy(c.pool.data))
    return c


@pytest.mark.parametrize("heads", [(8, 8, 128, 8), (8, 8, 256, 8)])
def test_values_that_cancel_over_a_long_piece(heads):
    """Equal weights over 131072 values whose mean is zero, by one workgroup (512 units): what the sums of codes and of their offset
    leave. q is zero, so P is 1 and P s exact; a token's value is s (c - 8) + z, each has a partner with 16 - c and -z."""
    def pool(c, ids):
        shape = c.pool.codes()[ids].shape
        nib = c.rng.integers(1, 16, (len(ids) // 2,) + shape[1:-1] + (c.HD,), dtype=np.uint8)
        for at, x in ((ids[0::2], nib), (ids[1::2], 16 - nib)):
            c.pool.codes()[at] = x[..., 0::2] | x[..., 1::2] << 4
        half = c.pool.data[..., c.page * c.HD // 2:].view(np.float16)
        par = half.reshape(half.shape[:-1] + (c.page // 4, 4, 2, 4))
        s, z = (c.rng.uniform(a, b, (len(ids) // 2,) + par.shape[1:-2] + (4,)).astype(np.float16) for a, b in ((0.25, 0.4), (-0.5, 0.5)))
        for at, sign in ((ids[0::2], 1), (ids[1::2], -1)):
            par[at, ..., 0, :], par[at, ..., 1, :] = s, sign * z

    c = shared_pages([(131071, 1)] * 64, heads, 16, seed=16, pool=pool)
    c.dq.zero_()
    got = c.attention().astype(np.float64)
    # a wave's 32768 keys are 128 segments of 8 steps. Within one, codes of 16 + c sum up to 24 s 256 < 2^12, so a step's rounding is
    # 2^-13 at most, 2^-13.8 in the root mean square where it is 2 roundings; 1024 of them of 4 waves are 2^6 times as much: 2^-7.8 on 131072 keys, 2^-24.8.
    # Seven times that, and the output's own step. (Sums over all of a piece would leave 2^7 times as much.)
    assert np.abs(got).max() <= 7 * 2 ** -24.8 + 2 ** -25


@pytest.mark.parametrize("seqs,heads", [([(4000, 1)], MODEL), ([(4090, 5)], H8), ([(800, 3200)], H16), ([(3000, 700)] * 2, (16, 1, 128, 8))])
def test_one_heavy_token_of_no_value_and_many_light_ones(seqs, heads):
    """A first token whose weight is 2^12 times another's and whose value is zero, before thousands of small values: each product P s
    of the others is 2^-12 of a scale of 2^-9, and the output is their mean."""
    c = Call(seqs, heads, 64, False, seed=17)
    u = c.rng.choice([-1.0, 1.0], c.HD)
    for b in range(len(seqs)):
        t = np.arange(c.lens[b])
        for h in range(c.HK):
            k, v = 0.02 * c.rng.standard_normal((len(t), c.HD)), 0.006 * c.rng.standard_normal((len(t), c.HD))
            k[0], v[0] = u * (12 * np.log(2) / np.sqrt(c.HD)), 0
            for w, x in ((0, k), (1, v)):
                c.pool.put_rows(c.table[b, t // 64], t % 64, h, w, x)
    c.dpool.copy_(c.torch.from_numpy(c.pool.data))
    c.q[:] = u  # its score is sqrt(HD) |k| = 12 log 2, the others' 0.3 at most
    c.dq = c.torch.from_numpy(c.q).to("cuda:0")
    rows = {int(t) for b in range(len(seqs)) for t in (c.start[b + 1] - 1, c.start[b + 1] - 3) if t >= c.start[b]}
    got, want = c.attention(), c.expected(rows=rows)
    e = np.stack([got[t].astype(np.float64) - want[t] for t in sorted(want)])
    w = np.stack([want[t] for t in sorted(want)])
    # as check(), and the output's own steps of 2^-24
    assert np.isfinite(e).all() and np.linalg.norm(e) <= 2 ** -10 * np.linalg.norm(w) + 2 ** -25 * np.sqrt(e.size)


@pytest.mark.parametrize("seqs,heads", [
    ([(3000, 1)], MODEL), ([(20000, 1)], (16, 1, 128, 8)), ([(2000, 61)], MODEL), ([(1500, 5), (0, 40), (700, 1)], H8), ([(90, 1)] * 140, H16)])
def test_outputs_of_few_columns_are_rounded_once(seqs, heads):
    """P and its products with scales keep 22 bits, so what differs from the rounded exact output is rounding the other way."""
    c = Call(seqs, heads, 64, seed=18)
    want = c.expected(rows=some(c, 20))
    got = c.attention()
    w = np.stack([want[t] for t in sorted(want)])
    e = np.stack([got[t].astype(np.float64) for t in sorted(want)]) - w.astype(np.float16)
    # The largest error is a score's: sums near 2^13 (1032 times the sum of 32 of q) of four groups, rounded some four times to 2^-12 at most,
    # times a scale of 2^-1.6 and 1 / sqrt(HD) = 2^-4 (2^-3.5): 2^-16 of P, and of the output. Where an output lies within that of the
    # middle between two f16, it is a step off: in the mean, squared, a step (2^-10.5 of the value) times the error, 2^-26.5, of which the
    # root is 2^-13.2. (One f16 for P or P s: 2^-12.)
    assert np.linalg.norm(e) <= 2 ** -12.8 * np.linalg.norm(w)


# a sequence of many rows whose context is far longer than the others' (csrc/kv_attn.hip, limit_of) is cut into pieces beside blocks
# of many columns: in a ragged batch, among rows of equal numbers, by the plan of more than 128 sequences; also where it does not fit
@pytest.mark.parametrize("seqs,heads", [
    ([(9000, 40), (0, 900), (5, 1), (0, 900), (0, 900)], H16),
    ([(0, 800)] * 3 + [(9000, 800)], H16),
    ([(20, 1)] * 70 + [(0, 1000), (9000, 35), (0, 1000)] + [(3, 2)] * 60 + [(0, 900)], H16),
    ([(0, 1100), (6000, 50), (0, 1100), (0, 1000)], (16, 2, 128, 128)),
    ([(0, 3000)] + [(30, 20)] * 130, H16)])
def test_a_far_longer_context_among_many_rows(seqs, heads):
    c = Call(seqs, heads, 64, seed=19, extra=3)
    got = c.attention()
    check(got[:c.T], c.expected(rows=some(c, 20)))
    assert np.isfinite(got[:c.T]).all() and (got[c.T:] == 7).all()
    np.testing.assert_array_equal(c.attention().view(np.uint16), got.view(np.uint16))
    b = max(range(len(seqs)), key=lambda b: seqs[b][0])
    c.dev[1][b] = seqs[b][1] - 1
    bad = c.attention()
    mine = np.zeros(len(got), bool)
    mine[c.start[b]:c.start[b + 1]] = True
    assert np.isnan(bad[mine]).all()
    check(bad, {t: w for t, w in c.expected(rows=some(c, 20)).items() if not mine[t]})


# append with four passes a wave (csrc/kv.hip: n_rows (HQ + 2 HK) HD / 512 of 32768 and more), in a grid and in a list
@pytest.mark.parametrize("seqs", [[(0, 1100), (33, 1003), (250, 1100)], [(7, 3000), (0, 0)] + [(30, 1)] * 60 + [(5, 90)]])
@pytest.mark.parametrize("heads,f32", [((16, 16, 128, 128), False), ((16, 16, 128, 8), True), ((16, 4, 256, 64), True), ((8, 8, 256, 0), False)])
def test_append_with_four_passes(seqs, heads, f32):
    c = Call(seqs, heads, 32, not f32, f32, seed=20, extra=1)
    assert c.n_rows * (c.HQ + 2 * c.HK) * c.HD // 512 >= 32768
    check_append(c, *c.append())


# contexts whose pieces are cut and longer than 1024 keys, so that a wave loads page ids and starts its fetches anew within a piece
# that does not begin at key 0; the last two by a plan
@pytest.mark.parametrize("n,len,heads", [
    (16, 5120, (8, 8, 256, 64)), (16, 5120, (8, 8, 128, 8)), (7, 20480, (4, 4, 256, 64)), (131, 5120, (4, 1, 256, 64)), (131, 5120, (3, 1, 128, 8))])
def test_cut_pieces_of_more_than_1024_keys(n, len, heads):
    c = shared_pages([(len - 1, 1)] * n, heads, 8, seed=21)
    keys = -(-n * heads[1] * len // (512 * 128)) * 128  # of a piece, as the device shares the work out
    assert 1024 < keys < len - 128
    check(c.attention(), c.expected(rows={0, n // 2, n - 1}))


# equal numbers of rows, laid out in a grid of (sequence, KV head) pairs (contexts of at most twice the rows)
@pytest.mark.parametrize("seqs,heads", [([(300, 800)] * 4, (16, 2, 128, 128)), ([(100, 1400)] * 4, MODEL), ([(0, 1000)] * 3, (32, 4, 128, 64))])
def test_equal_numbers_of_rows(seqs, heads):
    c = Call(seqs, heads, 32, seed=22)
    assert c.n_rows == len(seqs) * c.max_rows and c.max_len <= 2 * c.max_rows
    full = c.attention()
    check(full, c.expected(rows=some(c, 20)))
    # the same bounds with fewer rows, shorter contexts and a sequence that does not fit
    n = [c.max_rows, c.max_rows - 77, 5, 130][:len(seqs)]
    c.start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    c.lens = np.array([c.lens[0], c.max_rows, 4, 400][:len(seqs)], np.int32)
    c.T = int(c.start[-1])
    c.dev[0].copy_(c.torch.from_numpy(c.start))
    c.dev[1].copy_(c.torch.from_numpy(c.lens))
    got = c.attention()
    bad = set(range(c.start[2], c.start[3]))
    assert np.isnan(got[sorted(bad)]).all() and (got[c.T:] == 7).all()
    check(got[:c.T], {t: w for t, w in c.expected(rows=some(c, 20) - bad).items()})


@pytest.mark.parametrize("seqs,heads", [([(300, 3), (40, 1)], MODEL), ([(2000, 1)], H8), ([(0, 3000)], H16), ([(0, 800)] * 4, H8)])
def test_scores_in_the_hundreds(seqs, heads):
    """Scores of up to 400: one key takes nearly all, and maxima rise by more than P may."""
    c = Call(seqs, heads, 16, seed=23)
    c.q[:] = c.q * np.float16(40)
    c.dq = c.torch.from_numpy(c.q).to("cuda:0")
    want = c.expected(rows=some(c, 60))
    got = c.attention()
    e = np.stack([got[t].astype(np.float64) - want[t] for t in sorted(want)])
    w = np.stack([want[t] for t in sorted(want)])
    # q and the codes are exact, so a score's error is that of f32 sums near 1032 times the sum of 32 of q (2^17.8, a rounding 2^-6 at most and
    # 2^-6.8 in the root mean square), four of them in each of four groups, times a scale of 2^-1.6 (2^-2 for groups of 32 channels) and
    # 1 / sqrt(HD): 2^-10.4, 2^-10.3 for HD 128. It moves an output between two values, at most once its norm: 2^-9 with P's and the
    # output's roundings.
    assert np.isfinite(e).all() and np.linalg.norm(e) <= 2 ** -9 * np.linalg.norm(w)


@pytest.mark.parametrize("seqs,heads,f32", [([(700, 1), (40, 6), (0, 30)], MODEL, False), ([(0, 700), (9, 1)], H16, False), ([(20, 7), (300, 5)], H8, True)])
def test_offsets_beyond_32_bits(seqs, heads, f32):
    """Pages behind the first 4 GiB of a pool, and fused rows 512 MiB apart: the bits of the same calls nearby."""
    c = Call(seqs, heads, 64, True, f32, seed=24)
    t = c.torch
    q, v, pool = c.append()
    want = c.attention(q=t.from_numpy(q).to("cuda:0"))
    far = (1 << 32) // c.dpool[0].numel() + 5
    big = t.empty((far + c.n_pages,) + tuple(c.dpool.shape[1:]), dtype=t.uint8, device="cuda:0")
    big[far:].copy_(t.from_numpy(c.pool.data))
    kv = ha.PagedKV(big, far + c.n_pages, page_size=64, max_ctx=c.max_len, HQ=c.HQ, HK=c.HK, HD=c.HD, rot_dim=c.rot, dtype=ha.F32 if f32 else ha.F16)
    kv.set_param(0, "q_norm", c.qw)
    kv.set_param(0, "k_norm", c.kw)
    table = t.where(c.dev[2] >= 0, c.dev[2] + far, c.dev[2])
    b = c.make_batch(pages=table)
    n = min(c.n_rows, 12)
    rows, stride = c.drows, c.stride
    if n == c.n_rows:  # (few rows: far apart as well)
        stride = (1 << 29) // c.drows.element_size()
        rows = t.empty(n * stride, dtype=c.drows.dtype, device="cuda:0").view(n, stride)
        rows[:, :c.stride].copy_(c.drows)
    dq, dv = t.full_like(c.dq, 7.0), t.full((c.n_rows, 2, c.HK, c.HD), 7.0, dtype=t.float16, device="cuda:0")
    out = t.full_like(c.dq, 7.0)
    kv.append(0, b, rows, stride, dq, dv)
    kv.attention(0, b, dq, rows, stride, out)
    t.cuda.synchronize()
    for got, x in ((dq, q), (dv, v), (out, want)):
        np.testing.assert_array_equal(got.cpu().numpy().view(np.uint16), x.view(np.uint16))
    np.testing.assert_array_equal(big[far:].cpu().numpy(), pool)
    kv.close()
