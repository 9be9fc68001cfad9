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


BUFFERS = r"""
const path = require('path');
const ha = require(path.join(%(js)r, 'engine.js'));
const buffer = (bytes) => Object.assign(Object.create(ha.DeviceBuffer.prototype), {bytes: bytes, ptr: BigInt(4096), _borrows: 0});
const code = (fn) => { try { return fn(); } catch (e) { return e.name + ': ' + e.message; } };
const kv = Object.assign(Object.create(ha.PagedKV.prototype), {engine: null, _h: {}, config: {HQ: 4, HK: 2, HD: 128, gated: 1, dtype: %(dtype)d}});
const width = 4 * 2 * 128 + 2 * 2 * 128, stride = width + 64, e = %(dtype)d ? 2 : 4;
const need = {rows: e * (2 * stride + width), q: 2 * 3 * 4 * 128, values: 2 * 3 * 2 * 2 * 128, out: 2 * 3 * 4 * 128, rowStart: 12, lens: 8, pages: 32};
const out = {};
for (const less of [null].concat(Object.keys(need))) {
  const at = (k) => k === less ? (k.length & 1 ? buffer(need[k] - 1) : new ha.DeviceView(buffer(need[k] + 4), 8)) : buffer(need[k]);
  const b = {nSeqs: 2, nRows: 3, maxRows: 2, maxLen: 20, tableStride: 4, rowStart: at('rowStart'), lens: at('lens'), pages: at('pages')};
  out[less] = [code(() => kv.append(0, b, at('rows'), stride, at('q'), at('values'))), code(() => kv.append(0, b, at('rows'), stride, null, null)),
               code(() => kv.attention(0, b, at('q'), at('rows'), stride, at('out')))];
}
console.log(JSON.stringify(out));
"""


@pytest.mark.parametrize("dtype", [0, 1])
def test_buffers_that_end_too_early(dtype):
    """Each buffer of a call one byte (a view: one element) short; a call that gets past that has no handle."""
    r = subprocess.run([NODE, "-e", BUFFERS % {"js": JS, "dtype": dtype}], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    out = json.loads(r.stdout.strip().splitlines()[-1])
    handle = "TypeError: not a PagedKV handle"
    reach = {"null": (), "rows": (0, 1, 2), "q": (0, 2), "values": (0,), "out": (2,), "rowStart": (0, 1, 2), "lens": (0, 1, 2), "pages": (0, 1, 2)}
    for name, calls in reach.items():
        for i in range(3):
            want = "RangeError: %s of " % name if i in calls else handle
            assert out[name][i].startswith(want), (name, i, out[name][i])
