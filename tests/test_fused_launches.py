"""What the products whose results are not stored as they are launch, on the CPU (tests/fused_launches.py)."""
import os

import pytest

from fused_launches import CXX, HIPCC, ask, fused, logprobs, put

pytestmark = pytest.mark.skipif(not (os.path.exists(HIPCC) and os.path.exists(CXX)), reason="hipcc is missing")
ROWS = [1, 2, 3, 16, 17, 33, 100, 1000, 65537, 1 << 20]


def parts(launches, M):
    """The launches take each of M rows once, in order."""
    assert sum(x.rows for x in launches) == M
    at = 0
    for x in launches:
        yield x, at
        at += x.rows


def small(x):
    return 0 < x.groups * x.threads < 1 << 32


def test_threads_of_products():
    """HIP takes launches of fewer than 2^32 threads: calls of more are parted by rows, or go to a kernel with fewer."""
    calls = [(M, N, K, fmt, gated, q_at) for M in ROWS for N in (2, 1000, 12288, 248320, 1 << 24, 1 << 27, (1 << 29) - 64, 1 << 30)
             for K in (32, 64, 2048, 2080, 4096) for fmt in ((4, 32, False), (3, 32, True)) for gated in (False, True) for q_at in (0, 2 * 4) if M * N <= 1 << 40]
    parted = 0
    for (M, N, K, fmt, gated, q_at), got in zip(calls, ask([fused(*c[:5], q_at=c[5]) for c in calls])):
        case = (M, N, K, fmt, gated, q_at)
        fast = K % 64 == 0 and (q_at == 0 or fmt[0] != 4)
        if N > (1 << 29) - 64 and not fast:
            assert got.status == -1 and "2^29" in got.refusal and not got.launches, case
            continue
        assert got.status == 0, (case, got)
        cols = N // 2 if gated else N
        for x, row in parts(got.launches, M):
            assert small(x), (case, x)
            assert (x.a, x.out, x.residual) == (row * K * 2, row * cols * 4, row * cols * 2), (case, x)
        parted += len(got.launches) > 1
    assert parted


def test_threads_of_log_probabilities():
    calls = [(M, V, K, fmt) for M in ROWS + [20000, 40000] for V in (1, 100, 5000, 32768, 32769, 248320, 1 << 20) for K in (32, 64, 256, 2080)
             for fmt in ((4, 32, False), (2, 64, True)) if K % fmt[1] == 0]
    parted = 0
    for (M, V, K, fmt), got in zip(calls, ask([logprobs(*c, targets=2, top_k=1) for c in calls])):
        case = (M, V, K, fmt)
        assert got.status == 0, (case, got)
        records = [x for x in got.launches if "logprobs_kernel" not in x.kernel]
        joins = [x for x in got.launches if "logprobs_kernel" in x.kernel]
        assert all(small(x) for x in got.launches), case
        for x, row in parts(joins, M):
            assert (x.groups, x.a, x.logp, x.lse, x.top_ids) == (x.rows, row * K * 2, row * 8, row * 4, row * 4), (case, x)
        for x, row in parts(records, M):
            assert x.a == row * K * 2 and (x.records < 0 or x.records == row * -(-V // 64) * 16), (case, x)
        parted += len(records) > len(joins)
    assert parted


def test_lds_limits_are_constants():
    """A kernel's limit on dynamic LDS is the function's, in every thread: a call that set one of its own could take it from another
    call's launch. So each kernel has one, which no launch exceeds."""
    calls = [logprobs(M, V, K, fmt, targets=T, top_k=k) for M in (1, 7, 16, 40, 300, 3000) for V in (64, 2000, 5000, 32768, 40000, 248320, 1 << 20)
             for K in (256, 2048, 4096, 8192) for T in (0, 1, 1024) for k in (0, 5, 64) for fmt in ((4, 32, False), (3, 64, True))]
    limits, most = {}, {}
    for got in ask(calls):
        assert got.status == 0
        for name, n in got.limits:
            limits.setdefault(name, set()).add(n)
        for x in got.launches:
            most[x.kernel] = max(most.get(x.kernel, 0), x.lds)
    assert len([n for n in most if "stream" in n and n in limits]) and len([n for n in most if "logprobs" in n and n in limits])
    for name, n in most.items():
        assert n <= 48 * 1024 or len(limits[name]) == 1 and n <= min(limits[name]) <= 128 * 1024, (name, n, limits[name])


def test_outputs_over_what_is_read():
    """Rows are written while others read a and the targets: an output that overlaps them by a value is refused, one that ends where
    they begin, or begins where they end, is not. logp may be the targets' own memory: a row reads its targets first."""
    M, K, T, k = 7, 96, 3, 5
    size = {"logp": 4 * M * T, "entropy": 4 * M, "lse": 4 * M, "top_ids": 4 * M * k, "top_logp": 4 * M * k}
    read = {"a": 2 * M * K, "targets": 4 * M * T}
    for V in (1000, 40000):
        for name, n in size.items():
            for base, m in read.items():
                call = logprobs(M, V, K, targets=T, top_k=k)
                at = {-n: True, -n + 4: False, 0: (name, base) == ("logp", "targets"), 4: False, m - 4: False, m: True}
                for (x, fine), got in zip(at.items(), ask([y for x in at for y in (put(name, base, x), call)])):
                    case = (V, name, base, x, got)
                    if fine:
                        assert got.status == 0 and len(got.launches) == 2, case
                    else:
                        assert got.status == -1 and "overlap" in got.refusal and not got.launches, case


def test_workspaces_serve_fewer_rows():
    """The bytes asked for M rows never fall with M, and are taken by every call of fewer rows, although small calls store logits
    where larger ones leave records of a sixteenth; stored logits are 1 GiB at most, in parts of the rows."""
    rows = [1, 2, 16, 64, 65, 127, 128, 129, 255, 256, 257, 300, 1000, 8192, 8193, 20000, 32640, 32641, 1 << 20]
    for V, k in [(1, 0), (255, 1), (1000, 3), (1000, 4), (5000, 5), (32000, 5), (32000, 22), (32000, 23), (32768, 0), (32768, 64), (32769, 64), (248320, 20)]:
        need = [x.bytes for x in ask([("bytes", M, V, 64, 0, 0, k) for M in rows])]
        assert need == sorted(need), (V, k, need)
        assert all(n <= max(1 << 30, M * -(-V // 64) * 16) for M, n in zip(rows, need)), (V, k)
        for M, got in zip(rows, ask([logprobs(M, V, 64, targets=1, top_k=k, workspace=need[-1]) for M in rows])):
            assert got.status == 0, (V, k, M, got.refusal)
        for i in range(1, len(rows)):
            for M, got in zip(rows[:i + 1], ask([logprobs(M, V, 64, targets=1, top_k=k, workspace=need[i]) for M in rows[:i + 1]])):
                assert got.status == 0, (V, k, M, rows[i], got.refusal)
                joins = [x for x in got.launches if "logprobs_kernel" in x.kernel]
                for x, row in parts(joins, M):
                    assert (x.a, x.logp, x.lse, x.top_ids) == (row * 128, row * 4, row * 4, row * 4 * k if k else 0), (V, k, M, x)
                    assert x.records >= 0 or x.out == 0 and x.rows * V * 4 <= min(need[i], 1 << 30), (V, k, M, x)
