"""The sizes of the GPU tests of products and log probabilities reach every kernel that is compiled, each in every format (on the CPU,
tests/fused_launches.py)."""
import os

import pytest

import test_gpu_fused_kernels as tk
import test_gpu_logprobs_records as tr
from fused_launches import CXX, HIPCC, ask, fused, kernels, logprobs

pytestmark = pytest.mark.skipif(not (os.path.exists(HIPCC) and os.path.exists(CXX)), reason="hipcc is missing")


def reached(calls, answers):
    """(kernel, group) of the launches."""
    out = set()
    for c, got in zip(calls, answers):
        assert got.status == 0 and got.launches, c
        out |= {(x.kernel, c[3][1]) for x in got.launches}
    return out


def test_every_kernel():
    products, scores = tk.cases(), tr.cases()
    there = reached(products, ask([fused(*c) for c in products])) | reached(scores, ask([logprobs(*c, targets=2, top_k=7 if c[1] != tr.V else 5) for c in scores]))
    assert kernels() - {k for k, _ in there} == set()
    one = {"fused_rows_kernel": -1, "fused_stream_kernel": -1, "fused_tiles_kernel": -1}  # (their last argument: groups of 64 as one sum)
    for k in kernels():
        name, args = k[:-1].split("<")
        groups = {g for x, g in there if x == k}
        whole = name in one and args.split(", ")[-1] == "1"
        pair = name in one and any(x == k[:-2] + "1>" for x in kernels())  # (another kernel takes groups of 64)
        assert groups == ({64} if whole else {32} if pair else {32, 64}), (k, groups)


def test_where_the_records_are():
    """Every size of the tests of records leaves records, by the kernel that the test means."""
    sizes = [(M, tr.V, K) for M, K in tr.SIZES + tr.SOME]
    kinds = set()
    for c, got in zip(sizes, ask([logprobs(*c, top_k=40) for c in sizes])):
        first = got.launches[0]
        assert first.records == 0 and first.out < 0, c
        name, args = first.kernel[:-1].split("<")
        kinds.add((name, *args.split(", ")[3:5]))
        assert ("any" in name) == (c[2] == 96) and ("stream" in name) == (c[0] <= 16 and c[2] % 256 == 0), (c, first)
    assert {x[1:] for x in kinds if x[0] == "fused_tiles_kernel"} == {("1", "1"), ("2", "1"), ("3", "1"), ("4", "1"), ("4", "2")}
