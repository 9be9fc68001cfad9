"""A torso whose projections add onto the residual stream and give the MLP's gated rows (Torso(fused=True)), and the log
probabilities that score() gives, at the widths and layers of the torso's own test: against the fp64 composition of the oracles
and the default torso, resumed from a cache, and bit for bit between the Python and the Node host."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import fused_ref as fr
import hybrid_attention as ha
import test_gpu_torso_model as tm
from test_gpu_logprobs import check
from test_gpu_torso_model import D, I, L0, L1, ROWS0, ROWS1, TYPES, VOCAB, mo

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TABLE = "layers.3.in_proj"  # 8256 rows of D values: a vocabulary other than the embedding's


def torso(model, fused):
    W, V, M = model
    t = tm._torso(W, V, M)
    t.fused = fused
    return t


@pytest.fixture(scope="module")
def model():
    return tm._model()


@pytest.fixture(scope="module")
def ids():
    return np.random.default_rng(5).integers(0, VOCAB, L0 + L1).astype(np.uint32)


def test_hidden_rows(model, ids):
    """Some twenty roundings to f16 (2^-11 each at most) lie between the embedding and a final row: in quadrature 1.3e-3; the
    bound is that of the default torso, which has nine more."""
    W, V, M = model
    t, plain = torso(model, True), torso(model, False)
    got, snaps = t.forward(ids[:L0], ROWS0, keep=True)
    more, _ = t.forward(ids[L0:], ROWS1, cache=snaps)
    full, _ = t.forward(ids, ROWS0 + [L0 + r for r in ROWS1])
    default, _ = plain.forward(ids, ROWS0 + [L0 + r for r in ROWS1])
    ref = tm._oracle(W, V, M, ids, ROWS0 + [L0 + r for r in ROWS1])
    e = [mo.rel_err(x, y) for x, y in ((full, ref), (default, ref), (got, ref[:3]), (more, ref[3:]), (full, default))]
    print("fused %.1e, default %.1e, prefix %.1e, resumed %.1e, fused against default %.1e" % tuple(e))
    assert max(e) < 1e-2
    again, _ = t.forward(ids, ROWS0 + [L0 + r for r in ROWS1])
    assert np.array_equal(full, again)


def test_steps_and_layers(model, ids):
    """The residual stream that enters a layer is the default's within the roundings, and a profile names the steps there are."""
    t, plain = torso(model, True), torso(model, False)
    t.forward(ids, ROWS0, timestamps=True, debug_layers=True)
    plain.forward(ids, ROWS0, debug_layers=True)
    assert len(t.diag["layers"]) == len(TYPES) - 1 and t.diag["gpu_ms"] > 0
    for a, b in zip(t.diag["layers"], plain.diag["layers"]):
        assert mo.rel_err(a, b) < 1e-2
    assert set(plain.profile(ids)) - set(t.profile(ids)) == {"silu", "bias"}


def test_no_rows_and_one_row(model, ids):
    t = torso(model, True)
    out, _ = t.forward(ids[:1], [0])
    assert out.shape == (1, D) and np.isfinite(out).all()
    out, snaps = t.forward(ids[:1], [], keep=True)
    assert out.shape == (0, D) and snaps
    s, _ = t.score(ids[:1], [], targets=np.zeros((0, 2), np.int32), top_k=2)
    assert s["logp"].shape == (0, 2) and s["entropy"].shape == (0,) and s["top_ids"].shape == (0, 2)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("table,n_vocab,scale", [("embed", 0, 0.0), (TABLE, 8191, 0.5)])
def test_score(model, ids, fused, table, n_vocab, scale):
    """Against 64 bits over the final norm's rows in f16, as forward gives them."""
    t = torso(model, fused)
    words, s, N, K = model[0][table]
    Wt = mo.dequant(words, s, N, K)[:n_vocab or N]
    rows = [0, 3, 17, 39, 40, 48]
    targets = np.random.default_rng(3).integers(0, len(Wt), (len(rows), 2)).astype(np.int32)
    targets[0, 1] = -1
    hidden, _ = t.forward(ids, rows)
    got, snaps = t.score(ids, rows, targets, 4, n_vocab, scale, table, keep=True, timestamps=True)
    assert snaps and t.diag["gpu_ms"] > 0
    want = fr.logprobs(hidden.astype(np.float16), Wt, scale or 1.0, targets, 4)
    got = dict(got, ids=got["top_ids"], top=got["top_logp"])
    check(got, want, 2, 4)


def test_score_resumed_and_all_rows(model, ids):
    t = torso(model, True)
    _, snaps = t.forward(ids[:L0], [], keep=True)
    hidden, _ = t.forward(ids[L0:], cache=snaps)
    got, _ = t.score(ids[L0:], top_k=2, cache=snaps)
    words, s, N, K = model[0]["embed"]
    assert got["lse"].shape == (L1,) and got["logp"].shape == (L1, 0)
    check(dict(got, ids=got["top_ids"], top=got["top_logp"]), fr.logprobs(hidden.astype(np.float16), mo.dequant(words, s, N, K), k=2), 0, 2)


def test_score_refusals(model, ids):
    t = torso(model, False)
    for bad in (np.zeros((2, 1), np.float32), np.zeros(2, np.int32), np.zeros((3, 1), np.int32), np.full((2, 1), 2 ** 31)):
        with pytest.raises(ValueError):
            t.score(ids, [0, 1], bad)
    with pytest.raises(ValueError):
        t.score(ids, [0], table="layers.0.down")
    with pytest.raises(ha.HAError):
        t.score(ids, [0], top_k=65)
    with pytest.raises(KeyError):
        t.score(ids, [0], table="head")


@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
def test_node(model, ids, tmp_path):
    import torch
    d, (W, V, Mx) = str(tmp_path), model
    rng = np.random.default_rng(8)
    M, stride = 5, D + 24
    a, x = rng.standard_normal((M, D)).astype(np.float16), rng.standard_normal((M, stride)).astype(np.float32)
    targets = rng.integers(0, 990, (len(ROWS1), 3)).astype(np.int32)
    ask = {"topK": 6, "nVocab": 990, "scale": 0.75}
    spec = {"types": TYPES, "D": D, "I": I, "rows0": ROWS0, "rows1": ROWS1, "weights": {k: {"N": v[2], "K": v[3]} for k, v in W.items()},
            "vectors": sorted(V), "mixer": [[i, k] for i, k, _ in Mx], "ask": ask, "table": "embed", "M": M, "stride": stride}
    for name, (words, s, _, _) in W.items():
        words.tofile(os.path.join(d, "w_%s.q" % name))
        s.tofile(os.path.join(d, "w_%s.s" % name))
    for name, v in V.items():
        v.tofile(os.path.join(d, "v_%s.bin" % name))
    for i, k, v in Mx:
        v.tofile(os.path.join(d, "m_%d_%s.bin" % (i, k)))
    for name, v in (("ids0", ids[:L0]), ("ids1", ids[L0:]), ("targets", targets), ("a", a), ("residual", x)):
        v.tofile(os.path.join(d, name + ".bin"))
    with open(os.path.join(d, "spec.json"), "w") as f:
        json.dump(spec, f)
    print("node fused torso: L0=%d L1=%d" % (L0, L1), flush=True)
    r = subprocess.run([shutil.which("node"), os.path.join(ROOT, "tests", "js", "napi_fused.js"), d], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    info = json.loads(r.stdout.strip().splitlines()[-1])
    assert info["gpu_ms"] > 0 and "gate_up" in info["profile"] and "silu" not in info["profile"] and "bias" not in info["profile"]

    def same(name, want):
        got = np.fromfile(os.path.join(d, name + ".bin"), want.dtype).reshape(want.shape)
        assert got.tobytes() == np.ascontiguousarray(want).tobytes(), name

    t = torso(model, True)
    h0, snaps = t.forward(ids[:L0], ROWS0, keep=True)
    h1, _ = t.forward(ids[L0:], ROWS1, cache=snaps)
    same("hidden0", h0)
    same("hidden1", h1)
    s, _ = t.score(ids[L0:], ROWS1, targets, ask["topK"], ask["nVocab"], ask["scale"], cache=snaps)
    for k, name in (("logp", "logp"), ("entropy", "entropy"), ("lse", "lse"), ("top_ids", "topIds"), ("top_logp", "topLogp")):
        same("s_" + name, s[k])
    up = lambda v: torch.from_numpy(v).to("cuda:0")  # noqa: E731
    da, dx = up(a), up(x)
    gated = torch.empty(M, I, dtype=torch.float16, device="cuda:0")
    torch.cuda.synchronize()
    t.w["layers.0.gate_up"].fused(M, da, gated, ha.Epilogue("silu", gated=True))
    o = t.w["layers.0.out_proj"]
    o.fused(M, da, dx, ha.Epilogue("gelu", bias=t.v["final_norm"], residual=dx, residual_stride=stride, out_dtype=ha.F32, out_stride=stride))
    e, top, tl = (torch.empty(M, n, dtype=dt, device="cuda:0") for n, dt in ((1, torch.float32), (3, torch.int32), (3, torch.float32)))
    p = ha.LogProbs(top_k=3, entropy=e, top_ids=top, top_logp=tl)
    o.logprobs(M, da, p, torch.empty(o.logprobs_bytes(M, p), dtype=torch.uint8, device="cuda:0"))
    torch.cuda.synchronize()
    same("gated", gated.cpu().numpy())
    same("onto", dx.cpu().numpy())
    same("entropy", e[:, 0].cpu().numpy())
    same("top", top.cpu().numpy())
