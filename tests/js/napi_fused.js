'use strict';
// Drives what the Node host builds on products that go straight into what follows (strands-decider-web_amd/js/engine.js): a
// Torso with opts.fused (a prefix forward that keeps its cache, a resumed one, a profile), its score(), and MatMulNBits.fused
// and logprobs by themselves. Files in the directory named by the first argument:
//   spec.json {types, D, I, rows0, rows1, weights: {name: {N, K}}, vectors: [names], mixer: [[i, name]...], ask: {topK, nVocab,
//   scale}, table, M, stride}, w_<name>.q / .s, v_<name>.bin, m_<i>_<name>.bin, ids0.bin / ids1.bin (u32), targets.bin (i32),
//   a.bin (f16 [M][D]), residual.bin (f32 [M][stride])
// and writes hidden0.bin, hidden1.bin, s_<logp|entropy|lse|topIds|topLogp>.bin, gated.bin (f16), onto.bin (f32), entropy.bin,
// top.bin; prints {gpu_ms, profile}.
const fs = require('fs');
const path = require('path');
const ha = require(path.join(__dirname, '..', '..', 'strands-decider-web_amd', 'js', 'engine.js'));

const dir = process.argv[2];
const spec = JSON.parse(fs.readFileSync(path.join(dir, 'spec.json'), 'utf8'));
const raw = (f) => { const b = fs.readFileSync(path.join(dir, f)); return b.buffer.slice(b.byteOffset, b.byteOffset + b.byteLength); };
const save = (f, x) => fs.writeFileSync(path.join(dir, f), Buffer.from(x.buffer, x.byteOffset, x.byteLength));
const u32 = (f) => Array.from(new Uint32Array(raw(f)));

const torso = new ha.Torso({ layer_types: spec.types, hidden_size: spec.D, intermediate_size: spec.I }, { fused: true });
const lead = torso.lead, keep = [];
const up = (f) => { const x = new Uint8Array(raw(f)), b = lead.alloc(x.byteLength).upload(x); keep.push(b); return b; };
const take = (bytes) => { const b = lead.alloc(bytes); keep.push(b); return b; };
Object.keys(spec.weights).forEach((name) => torso.setWeight(name,
  Object.assign({ q: up('w_' + name + '.q'), s: up('w_' + name + '.s') }, spec.weights[name])));
spec.vectors.forEach((name) => torso.setParam(name, new Float32Array(raw('v_' + name + '.bin'))));
spec.mixer.forEach(([i, name]) => torso.setParam('layers.' + i + '.' + name, new Float32Array(raw('m_' + i + '_' + name + '.bin'))));

const r0 = torso.forward(u32('ids0.bin'), spec.rows0, { keepCache: true });
const r1 = torso.forward(u32('ids1.bin'), spec.rows1, { cache: r0.cache });
save('hidden0.bin', r0.hidden);
save('hidden1.bin', r1.hidden);
const flat = new Int32Array(raw('targets.bin')), T = flat.length / spec.rows1.length;
const targets = spec.rows1.map((_, i) => Array.from(flat.slice(i * T, (i + 1) * T)));
const ask = Object.assign({ targets: targets, table: spec.table }, spec.ask);
const s = torso.score(u32('ids1.bin'), spec.rows1, ask, { cache: r0.cache, timestamps: true });
['logp', 'entropy', 'lse', 'topIds', 'topLogp'].forEach((k) => save('s_' + k + '.bin', s[k]));
const none = torso.score(u32('ids1.bin'), [], Object.assign({}, ask, { targets: [] }), { cache: r0.cache });
if (none.entropy.length !== 0 || s.hidden !== undefined) throw new Error('score of no rows');
const plain = torso.score(u32('ids1.bin'), spec.rows1, { table: spec.table, nVocab: spec.ask.nVocab, scale: spec.ask.scale },
  { cache: r0.cache });
if (plain.logp.length !== 0 || plain.topIds.length !== 0 || plain.lse.some((x, i) => x !== s.lse[i])) throw new Error('score without targets');
r0.cache.release();
const profile = torso.profile(u32('ids0.bin'));

const M = spec.M, D = spec.D, w = torso.weights['layers.0.gate_up'].h, o = torso.weights['layers.0.out_proj'].h;
const a = up('a.bin'), x = up('residual.bin'), gated = take(2 * M * w.N / 2);
w.fused(M, a, gated, { act: 'silu', gated: true });
o.fused(M, a, new ha.DeviceView(x, 0), { act: 'gelu', bias: torso.vectors.final_norm, residual: x, residualStride: spec.stride,
  outDtype: ha.F32, outStride: spec.stride });
save('gated.bin', gated.download(new Uint8Array(gated.bytes)));
save('onto.bin', x.download(new Uint8Array(x.bytes)));
const entropy = take(4 * M), ids = take(4 * M * 3), top = take(4 * M * 3);
const p = { topK: 3, entropy: entropy, topIds: ids, topLogp: top };
const work = take(o.logprobsBytes(M, p));
o.logprobs(M, a, p, work);
save('entropy.bin', entropy.download(new Float32Array(M)));
save('top.bin', ids.download(new Int32Array(3 * M)));
[() => o.logprobs(M, a, p, new ha.DeviceView(work, 16)), () => o.logprobs(M, a, { topK: 65, topIds: ids, topLogp: top }, work),
  () => o.fused(M, a, gated, { act: 'gelu', gated: true, residual: gated, residualStride: 8, residualDtype: ha.F16 }),
  () => o.fused(-1, a, gated, {})].forEach((fn, i) => {
  let got = 'nothing';
  try { fn(); } catch (e) { got = e.code || e.name; }
  if (got !== ['HA_1', 'RangeError', 'HA_1', 'HA_1'][i]) throw new Error('refusal ' + i + ': ' + got);
});
torso.dropWeights();
keep.forEach((b) => b.free());
torso.destroy();
console.log(JSON.stringify({ gpu_ms: s.gpu_ms, profile: profile }));
