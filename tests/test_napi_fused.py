"""MatMulNBits.fused and logprobs of the Node host without a GPU: what the addon refuses, and buffers that end too early."""
import json
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
JS = os.path.join(ROOT, "strands-decider-web_amd", "js")
NODE = shutil.which("node")
pytestmark = pytest.mark.skipif(NODE is None or not os.path.exists(os.path.join(JS, "ha_napi.node")), reason="node or the built addon is missing")


def node(script):
    r = subprocess.run([NODE, "-e", "const JS = %r;\n" % JS + script], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    return json.loads(r.stdout.strip().splitlines()[-1])


REFUSALS = r"""
const ha = require(JS + '/engine.js');
const nat = require(JS + '/ha_napi.node');
const code = (fn) => { try { return fn(); } catch (e) { return e.name + ': ' + e.message; } };
const p = BigInt(4096);
const w = Object.assign(Object.create(ha.MatMulNBits.prototype), {engine: null, _h: {}, N: 64, K: 64});
console.log(JSON.stringify({
  handle: [code(() => nat.mnbFused({}, 1, p, {}, p, null)), code(() => nat.mnbLogprobs(null, 1, p, {}, p, 0, null)),
           code(() => nat.mnbLogprobsBytes(p, 1, {})), code(() => w.fused(1, p, p)), code(() => w.logprobsBytes(1, {}))],
  act: [code(() => w.fused(1, p, p, {act: 'relu'})), code(() => w.fused(1, p, p, {act: 'toString'}))],
  dtype: code(() => w.fused(1, p, p, {outDtype: 'bf16'})),
  bias: code(() => w.fused(1, p, p, {bias: 4096})),
  targets: code(() => w.logprobs(1, p, {nTargets: 1, targets: [1]}, p, 64)),
}));
"""


def test_refusals():
    out = node(REFUSALS)
    assert out["handle"] == ["TypeError: not a MatMulNBits handle"] * 5
    assert out["act"] == ["RangeError: act must be null, 'silu' or 'gelu'"] * 2
    assert out["dtype"] == "TypeError: unsupported dtype bf16"
    for k in ("bias", "targets"):
        assert out[k] == "TypeError: layer buffers must be DeviceBuffer or BigInt device pointers"


BUFFERS = r"""
const ha = require(JS + '/engine.js');
const buffer = (bytes) => Object.assign(Object.create(ha.DeviceBuffer.prototype), {bytes: bytes, ptr: BigInt(4096), _borrows: 0});
const code = (fn) => { try { return fn(); } catch (e) { return e.name + ': ' + e.message; } };
const N = 96, K = 64, M = 3, T = 2, k = 5, work = 1000;
const w = Object.assign(Object.create(ha.MatMulNBits.prototype), {engine: null, _h: {}, N: N, K: K});
const rows = (size, cols, stride) => size * ((M - 1) * stride + cols);
const need = {a: 2 * M * K, bias: 4 * N, dense: rows(2, N, N), far: rows(4, N, N + 7), gated: rows(2, N / 2, N / 2), half: rows(2, N / 2, N),
              targets: 4 * M * T, logp: 4 * M * T, entropy: 4 * M, lse: 4 * M, topIds: 4 * M * k, topLogp: 4 * M * k, workspace: work};
const out = {};
for (const less of [null].concat(Object.keys(need))) {
  const at = (x) => x === less ? (x.length & 1 ? buffer(need[x] - 1) : new ha.DeviceView(buffer(need[x] + 4), 8)) : buffer(need[x]);
  const p = {nTargets: T, topK: k};
  ['targets', 'logp', 'entropy', 'lse', 'topIds', 'topLogp'].forEach((x) => { p[x] = at(x); });
  out[less] = [
    code(() => w.fused(M, at('a'), at('dense'), {bias: at('bias'), residual: at('far'), residualStride: N + 7})),
    code(() => w.fused(M, at('a'), at('gated'), {gated: true, residual: at('half'), residualDtype: ha.F16, residualStride: N})),
    code(() => w.fused(0, at('a'), at('dense'), {bias: at('bias')})),
    code(() => w.logprobs(M, at('a'), p, at('workspace'), work)),
    code(() => w.logprobs(M, at('a'), {lse: at('lse')}, at('workspace'))),
  ];
}
console.log(JSON.stringify(out));
"""


def test_buffers_that_end_too_early():
    """Each buffer of a call one byte (a view: one element) short; a call that gets past that has no handle."""
    out = node(BUFFERS)
    reach = {"null": {}, "a": {0: "a", 1: "a", 3: "a", 4: "a"}, "bias": {0: "bias"}, "dense": {0: "out"}, "far": {0: "residual"},
             "gated": {1: "out"}, "half": {1: "residual"}, "lse": {3: "lse", 4: "lse"}, "workspace": {3: "workspace"}}
    for x in ("targets", "logp", "entropy", "topIds", "topLogp"):
        reach[x] = {3: x}
    assert set(out) == set(reach)
    for less, calls in reach.items():
        for i in range(5):
            want = "RangeError: %s of " % calls[i] if i in calls else "TypeError: not a MatMulNBits handle"
            assert out[less][i].startswith(want), (less, i, out[less][i])


SCORE = r"""
const ha = require(JS + '/engine.js');
const code = (fn) => { try { return fn(); } catch (e) { return e.name + ': ' + e.message; } };
const torso = (o) => Object.assign(Object.create(ha.Torso.prototype), {D: 64, unrotate: null, embedRows: null, fused: false,
  weights: {embed: {N: 96, K: 64, had: 0}, head: {N: 96, K: 64, had: 64}, wide: {N: 96, K: 128, had: 0}}}, o);
const t = torso({});
console.log(JSON.stringify([
  code(() => t.score([1], null, {table: 'none'})), code(() => t.score([1], null, {table: 'wide'})),
  code(() => t.score([1], null, {table: 'head'})), code(() => torso({unrotate: [1]}).score([1])),
  code(() => torso({embedRows: (x) => x}).score([1])), code(() => t.score([1, 2], null, {targets: [[1]]})),
  code(() => t.score([1, 2], null, {targets: [[1], [2, 3]]})), code(() => t.score([1, 2], [1], {targets: [[1.5]]})),
  code(() => t.score([1], null, {targets: [[4294967296]]}))]));
"""


def test_score_refusals():
    out = node(SCORE)
    for got, want in zip(out, ["Error: no tensor none", "RangeError: wide has rows", "Error: score: head reads", "Error: score: this torso",
                               "Error: score: the embedding"] + ["RangeError: targets must be"] * 4):
        assert got.startswith(want), (got, want)
