"""PagedKV of the Node host without a GPU: what it exports, the config that reaches the C ABI, and its refusals."""
import json
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
JS = os.path.join(ROOT, "strands-decider-web_amd", "js")
NODE = shutil.which("node")
pytestmark = pytest.mark.skipif(NODE is None or not os.path.exists(os.path.join(JS, "ha_napi.node")), reason="node or the built addon is missing")

SCRIPT = r"""
const path = require('path');
const ha = require(path.join(%(js)r, 'engine.js'));
const nat = require(path.join(%(js)r, 'ha_napi.node'));
const code = (fn) => { try { return fn(); } catch (e) { return (e.code || e.name) + ': ' + e.message; } };
const p = BigInt(4096);
const batch = {nSeqs: 1, nRows: 1, maxRows: 1, maxLen: 1, tableStride: 1, rowStart: p, lens: p, pages: p};
console.log(JSON.stringify({
  bytes: [ha.PagedKV.pageBytes({}), ha.PagedKV.pageBytes({pageSize: 16, HQ: 4, HK: 4, HD: 128})],
  config: code(() => new ha.PagedKV(null, p, {nPages: 4, pageSize: 48})),
  type: code(() => new ha.PagedKV(null, p, {nPages: 4, HQ: 'eight'})),
  dtype: code(() => new ha.PagedKV(null, p, {nPages: 4, dtype: 'bf16'})),
  none: code(() => nat.kvCreate(null, p, 0)),
  pages: code(() => new ha.PagedKV(null, BigInt(8), {nPages: 4})),
  number: code(() => nat.kvCreate({nPages: 4}, 4096, 0)),
  append: code(() => nat.kvAppend({}, 0, batch, p, 1, p, p, null)),
  attention: code(() => nat.kvAttention(null, 0, batch, p, p, 1, p, null)),
  param: code(() => nat.kvSetParam(1, 0, 'q_norm', new Float32Array(256))),
  destroy: code(() => nat.kvDestroy(undefined)),
}));
"""


def test_refusals():
    r = subprocess.run([NODE, "-e", SCRIPT % {"js": JS}], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    out = json.loads(r.stdout.strip().splitlines()[-1])
    assert out["bytes"] == [2 * 2 * 64 * 144, 4 * 2 * 16 * 80]
    assert out["config"].startswith("HA_1: page_size") and out["pages"].startswith("HA_1: pages")
    assert out["type"] == out["none"] == "TypeError: invalid cache config field"
    assert out["dtype"] == "TypeError: unsupported dtype bf16" and out["number"] == "TypeError: pages must be a BigInt"
    for k in ("append", "attention", "param", "destroy"):
        assert out[k] == "TypeError: not a PagedKV handle"
