'use strict';
// Drives the KV cache's launchers from files written by the Python test: node tests/js/run_kv.js <dir>
// <dir>/spec.json: {T, nHq, nKv, hd, page, pages, width, S, keep, files: [names of raw files]}; results as <name>.out
const fs = require('fs');
const path = require('path');
const { createQwen3Host } = require(path.join(__dirname, '..', '..', 'tabinfer_amd', 'host', 'qwen3-host.js'));

const dir = process.argv[2];
const s = JSON.parse(fs.readFileSync(path.join(dir, 'spec.json'), 'utf8'));
const { E, L } = createQwen3Host({ device: 0 }).engine;
const b = {};
const zeros = (bytes) => { const x = E.createBuffer(bytes); E.fillU32(x, 0, bytes / 4); return x; };
for (const f of s.files) {
  const data = fs.readFileSync(path.join(dir, f));
  b[f] = E.createBuffer(data.length);
  E.writeBuffer(b[f], 0, new Uint8Array(data.buffer, data.byteOffset, data.length));
}
const save = (name, buf, bytes) => fs.writeFileSync(path.join(dir, name + '.out'), Buffer.from(E.readBytes(buf, 0, bytes)));
const { T, nHq, nKv, hd, page, pages, width, S, keep } = s;

const rows = page * pages * nKv;
const pool = { kq: zeros(rows * hd), ks: zeros(rows * hd / 8), vq: zeros(rows * hd), vs: zeros(rows * hd / 8), page, pages };
const table = { buf: b.table, width, B: 2 };
const k = zeros(T * nKv * hd * 4), v = zeros(T * nKv * hd * 4), o = zeros(T * nHq * hd * 4);
L.kvWritePagedQ8(b.k, b.v, pool, table, b.seq, b.pos, T, nKv, hd);
L.kvReadPagedQ8(pool, table, b.seq, b.pos, k, v, T, nKv, hd);
save('k', k, T * nKv * hd * 4);
save('v', v, T * nKv * hd * 4);
L.attnPagedQ8(b.q, pool, table, b.lens, o, nHq, nKv, hd, 9, 2);
save('paged', o, 2 * nHq * hd * 4);

const kv = { kq: b.kc, ks: b.ks, vq: b.vc, vs: b.vs };
const mass = zeros(S * nKv * 4), where = zeros(S * nKv * 4);
L.attnWindowQ8(b.q, kv, o, T, 0, nHq, nKv, hd, 7, 2);
save('window', o, T * nHq * hd * 4);
L.attnMassQ8(b.q, kv, o, mass, T, 0, nHq, nKv, hd);
save('mass_attn', o, T * nHq * hd * 4);
save('mass', mass, S * nKv * 4);
L.kvEvictQ8(kv, mass, where, S, 0, keep, 2, 3, S, nKv, hd);
save('where', where, S * nKv * 4);
save('cut', mass, S * nKv * 4);
save('kc', b.kc, S * nKv * hd);
process.exit(0);
