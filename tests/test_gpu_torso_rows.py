"""A torso asked for the same row more than once, in both hosts: each time the row that a single request gives, bit for bit. And
its score over a vocabulary whose logits are not stored."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import fused_ref as fr
import test_gpu_torso_model as tm
from test_gpu_logprobs import check
from test_gpu_torso_model import D, I, TYPES, VOCAB

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROWS = [7, 3] + [7] * 4000 + [0, 3, 8, 8]  # more output rows than run at once


@pytest.fixture(scope="module")
def model():
    return tm._model()


@pytest.fixture(scope="module")
def ids():
    return np.random.default_rng(6).integers(0, VOCAB, 9).astype(np.uint32)


def node(d, W, V, Mx, ids, rows, fused, ask=None):
    """What tests/js/napi_rows.js makes of the model."""
    exe = shutil.which("node")
    if exe is None:
        pytest.skip("node is not installed")
    spec = {"types": TYPES, "D": D, "I": I, "rows": rows, "fused": fused, "ask": ask, "weights": {k: {"N": v[2], "K": v[3]} for k, v in W.items()},
            "vectors": sorted(V), "mixer": [[i, k] for i, k, _ in Mx]}
    for name, (words, s, _, _) in W.items():
        words.tofile(os.path.join(d, "w_%s.q" % name))
        s.tofile(os.path.join(d, "w_%s.s" % name))
    for name, v in V.items():
        v.tofile(os.path.join(d, "v_%s.bin" % name))
    for i, k, v in Mx:
        v.tofile(os.path.join(d, "m_%d_%s.bin" % (i, k)))
    ids.tofile(os.path.join(d, "ids.bin"))
    with open(os.path.join(d, "spec.json"), "w") as f:
        json.dump(spec, f)
    r = subprocess.run([exe, os.path.join(ROOT, "tests", "js", "napi_rows.js"), d], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    return lambda name, dtype: np.fromfile(os.path.join(d, name + ".bin"), dtype)


@pytest.mark.parametrize("fused", [False, True])
def test_rows(model, ids, fused, tmp_path):
    W, V, Mx = model
    t = tm._torso(W, V, Mx)
    t.fused = fused
    single, _ = t.forward(ids)
    scores, _ = t.score(ids, top_k=3)
    got, _ = t.forward(ids, ROWS)
    assert np.array_equal(got, single[ROWS])
    got, _ = t.score(ids, ROWS[:2] + ROWS[-4:], top_k=3)
    for n, x in got.items():
        assert np.array_equal(x, scores[n][ROWS[:2] + ROWS[-4:]]), n
    again, _ = t.forward(ids, [8, 8])
    assert np.array_equal(again, single[[8, 8]])
    read = node(str(tmp_path), W, V, Mx, ids, ROWS, fused)
    assert np.array_equal(read("hidden", np.float32).reshape(len(ROWS), D), single[ROWS])
    many, _ = t.score(ids, ROWS, top_k=3)
    assert np.array_equal(read("lse", np.float32), many["lse"])
    assert np.array_equal(read("topIds", np.int32).reshape(-1, 3), many["top_ids"])


@pytest.mark.parametrize("fused", [False, True])
def test_score_over_a_large_table(model, ids, fused, tmp_path):
    """A vocabulary whose logits are not stored, its last block cut, against 64 bits over the final norm's rows in f16."""
    W, V, Mx = model
    N, n_vocab, rows = 33000, 32901, [8, 0, 5, 5]
    words, s, _, table = fr.weight(N, D, seed=40, std=2 / np.sqrt(D))
    W = dict(W, head=(words, s, N, D))
    targets = np.random.default_rng(41).integers(0, n_vocab, (len(rows), 2)).astype(np.int32)
    t = tm._torso(W, V, Mx)
    t.fused = fused
    hidden, _ = t.forward(ids, rows)
    got, _ = t.score(ids, rows, targets, 5, n_vocab, 0.75, "head")
    want = fr.logprobs(hidden.astype(np.float16), table[:n_vocab], 0.75, targets, 5)
    check(dict(got, ids=got["top_ids"], top=got["top_logp"]), want, 2, 5)
    read = node(str(tmp_path), W, V, Mx, ids, rows, fused, {"topK": 5, "nVocab": n_vocab, "scale": 0.75, "table": "head", "targets": targets.tolist()})
    for n, name in (("lse", "lse"), ("top_ids", "topIds"), ("logp", "logp")):
        assert read(name, got[n].dtype).tobytes() == np.ascontiguousarray(got[n]).tobytes(), n
