'use strict';
// Drives the paged 4-bit K/V cache of the Node host (PagedKV, strands-decider-web_amd/js/engine.js): one batch appended to and
// attended in both layers, on the engine's stream. Files in the directory named by the first argument: spec.json {config, batch
// {nSeqs, nRows, maxRows, maxLen, tableStride}, rowStride}, rows.bin (f16), pages.bin, start.bin, lens.bin, table.bin (i32),
// w_<layer>_<q|k>.bin (f32 gains); writes pages_out.bin, q_<layer>.bin, values_<layer>.bin, out_<layer>.bin (f16).
const fs = require('fs');
const path = require('path');
const ha = require(path.join(__dirname, '..', '..', 'strands-decider-web_amd', 'js', 'engine.js'));

const dir = process.argv[2];
const spec = JSON.parse(fs.readFileSync(path.join(dir, 'spec.json'), 'utf8'));
const engine = ha.Engine.createSync({ layer_types: ['full_attention'] }, { batch: 1, maxCtx: 64 });

function read(file) {
  const buf = fs.readFileSync(path.join(dir, file));
  return new Uint8Array(buf.buffer, buf.byteOffset, buf.byteLength);
}
function upload(file) {
  const u8 = read(file);
  return engine.alloc(u8.byteLength).upload(u8);
}
function save(file, buf) {
  fs.writeFileSync(path.join(dir, file), Buffer.from(buf.download(new Uint8Array(buf.bytes)).buffer));
}
function expect(what, code, fn) {
  let got = 'nothing';
  try { fn(); } catch (e) { got = e.code || e.name; }
  if (got !== code) throw new Error(what + ': ' + got + ' instead of ' + code);
}

const c = spec.config;
const pages = upload('pages.bin');
if (pages.bytes !== ha.PagedKV.pageBytes(c) * c.nPages * c.nLayers) throw new Error('page bytes');
const kv = new ha.PagedKV(engine, new ha.DeviceView(pages, 0), c);
const bufs = ['start.bin', 'lens.bin', 'table.bin', 'rows.bin'].map(upload);
const batch = Object.assign({ rowStart: bufs[0], lens: bufs[1], pages: new ha.DeviceView(bufs[2], 0) }, spec.batch);
const n = spec.batch.nRows;
const q = engine.alloc(n * c.HQ * c.HD * 2), values = engine.alloc(n * 2 * c.HK * c.HD * 2), out = engine.alloc(n * c.HQ * c.HD * 2);
for (let i = 0; i < c.nLayers; i++) {
  ['q', 'k'].forEach((x) => {
    const w = read('w_' + i + '_' + x + '.bin');
    kv.setParam(i, x + '_norm', new Float32Array(w.buffer.slice(w.byteOffset, w.byteOffset + w.byteLength)));
  });
  kv.append(i, batch, bufs[3], spec.rowStride, q, values);
  kv.attention(i, batch, q, bufs[3], spec.rowStride, out);
  save('q_' + i + '.bin', q);
  save('values_' + i + '.bin', values);
  save('out_' + i + '.bin', out);
}
save('pages_out.bin', pages);
expect('a layer that is not there', 'HA_1', () => kv.append(c.nLayers, batch, bufs[3], spec.rowStride, q, null));
expect('rows that are too short', 'HA_1', () => kv.append(0, batch, bufs[3], spec.rowStride - 8 * c.HD, q, null));
expect('no gates', 'HA_1', () => kv.attention(0, batch, q, null, 0, out));
expect('a batch without arrays', 'HA_1', () => kv.attention(0, spec.batch, q, bufs[3], spec.rowStride, out));
expect('no Float32Array', 'TypeError', () => kv.setParam(0, 'q_norm', new Float64Array(c.HD)));
expect('too few pages', 'RangeError', () => new ha.PagedKV(engine, new ha.DeviceView(pages, 16), c));
expect('borrowed pages', 'HA_BORROWED', () => pages.free());
kv.destroy();
kv.destroy();  // idempotent
expect('a destroyed handle', 'TypeError', () => kv.append(0, batch, bufs[3], spec.rowStride, q, null));
bufs.concat([q, values, out, pages]).forEach((x) => x.free());
engine.destroy();
console.log(JSON.stringify({ ok: true }));
