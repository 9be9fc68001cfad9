'use strict';
// A Torso of the Node host asked for rows more than once. The directory named by the first argument holds the model as
// tests/js/napi_fused.js reads it (spec.json {types, D, I, rows, fused, weights, vectors, mixer}, w_<name>.q / .s, v_<name>.bin,
// m_<i>_<name>.bin, ids.bin); writes hidden.bin and, of its score (of spec.ask where there is one), lse.bin, topIds.bin, logp.bin.
const fs = require('fs');
const path = require('path');
const ha = require(path.join(__dirname, '..', '..', 'strands-decider-web_amd', 'js', 'engine.js'));

const dir = process.argv[2];
const spec = JSON.parse(fs.readFileSync(path.join(dir, 'spec.json'), 'utf8'));
const raw = (f) => { const b = fs.readFileSync(path.join(dir, f)); return b.buffer.slice(b.byteOffset, b.byteOffset + b.byteLength); };
const save = (f, x) => fs.writeFileSync(path.join(dir, f), Buffer.from(x.buffer, x.byteOffset, x.byteLength));

const torso = new ha.Torso({ layer_types: spec.types, hidden_size: spec.D, intermediate_size: spec.I }, { fused: spec.fused });
const keep = [], up = (f) => { const x = new Uint8Array(raw(f)), b = torso.lead.alloc(x.byteLength).upload(x); keep.push(b); return b; };
Object.keys(spec.weights).forEach((name) => torso.setWeight(name,
  Object.assign({ q: up('w_' + name + '.q'), s: up('w_' + name + '.s') }, spec.weights[name])));
spec.vectors.forEach((name) => torso.setParam(name, new Float32Array(raw('v_' + name + '.bin'))));
spec.mixer.forEach(([i, name]) => torso.setParam('layers.' + i + '.' + name, new Float32Array(raw('m_' + i + '_' + name + '.bin'))));
const ids = Array.from(new Uint32Array(raw('ids.bin')));
save('hidden.bin', torso.forward(ids, spec.rows).hidden);
const s = torso.score(ids, spec.rows, spec.ask || { topK: 3 });
['lse', 'topIds', 'logp'].forEach((k) => save(k + '.bin', s[k]));
torso.dropWeights();
keep.forEach((b) => b.free());
torso.destroy();
