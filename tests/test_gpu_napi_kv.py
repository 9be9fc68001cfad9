"""PagedKV of the Node host on the GPU: tests/js/napi_kv.js appends a ragged batch to two layers and attends it; pages, queries,
stored values and outputs equal those of the same calls through the C ABI from Python, bit for bit."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import hybrid_attention as ha

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")]
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HQ, HK, HD, PAGE, NP, LAYERS = 8, 2, 256, 16, 24, 2


def test_node_paged_kv(tmp_path):
    import torch
    rng = np.random.default_rng(11)
    new, lens = [37, 1, 20], np.array([60, 130, 20], np.int32)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    table = np.full((3, 10), -1, np.int32)
    ids = list(rng.permutation(NP))
    for b in range(3):
        table[b, :-(-lens[b] // PAGE)] = [ids.pop() for _ in range(-(-lens[b] // PAGE))]
    stride = HQ * 2 * HD + 2 * HK * HD + 8
    n = int(start[-1])
    rows = rng.standard_normal((n, stride)).astype(np.float16)
    nb = ha.PagedKV.page_bytes(PAGE, HK, HD)
    pages = rng.integers(0, 256, (LAYERS, NP, nb)).astype(np.uint8)
    # scales and zeros behind each block's codes: ordinary numbers (the pages a batch attends were written before it)
    blocks = pages.reshape(LAYERS, NP, HK, 2, -1)
    sz = blocks.shape[-1] - PAGE * HD // 2
    blocks[..., -sz:] = rng.uniform(0.1, 0.4, blocks.shape[:-1] + (sz // 2,)).astype(np.float16).view(np.uint8)
    w = rng.uniform(0.8, 1.2, (LAYERS, 2, HD)).astype(np.float32)
    d = str(tmp_path)
    for name, a in [("rows", rows), ("pages", pages), ("start", start), ("lens", lens), ("table", table)]:
        a.tofile(os.path.join(d, name + ".bin"))
    for i in range(LAYERS):
        for j, x in enumerate("qk"):
            w[i, j].tofile(os.path.join(d, "w_%d_%s.bin" % (i, x)))
    spec = {"config": {"nLayers": LAYERS, "nPages": NP, "pageSize": PAGE, "maxCtx": 160, "HQ": HQ, "HK": HK, "HD": HD},
            "batch": {"nSeqs": 3, "nRows": n, "maxRows": max(new), "maxLen": int(lens.max()), "tableStride": 10}, "rowStride": stride}
    with open(os.path.join(d, "spec.json"), "w") as f:
        json.dump(spec, f)
    print("node paged kv: %d rows" % n, flush=True)
    r = subprocess.run([shutil.which("node"), os.path.join(ROOT, "tests", "js", "napi_kv.js"), d], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert json.loads(r.stdout.strip().splitlines()[-1])["ok"]

    dev = "cuda:0"
    up = lambda x: torch.from_numpy(x).to(dev)  # noqa: E731
    pool = up(pages)
    kv = ha.PagedKV(pool, NP, page_size=PAGE, n_layers=LAYERS, max_ctx=160, HQ=HQ, HK=HK, HD=HD)
    batch = ha.KVBatch(3, n, max(new), int(lens.max()), up(start), up(lens), up(table), 10)
    dr = up(rows)
    q = torch.empty(n, HQ, HD, dtype=torch.float16, device=dev)
    out, values = torch.empty_like(q), torch.empty(n, 2, HK, HD, dtype=torch.float16, device=dev)

    def same(name, t):
        got = np.fromfile(os.path.join(d, name + ".bin"), np.uint8)
        np.testing.assert_array_equal(got, t.cpu().numpy().view(np.uint8).ravel(), name)

    for i in range(LAYERS):
        kv.set_param(i, "q_norm", w[i, 0])
        kv.set_param(i, "k_norm", w[i, 1])
        kv.append(i, batch, dr, stride, q, values)
        kv.attention(i, batch, q, dr, stride, out)
        torch.cuda.synchronize()
        for name, t in (("q", q), ("values", values), ("out", out)):
            same("%s_%d" % (name, i), t)
        assert torch.isfinite(out).all()
    same("pages_out", pool)
    kv.close()
