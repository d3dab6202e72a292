'use strict';
// Drives a served batch's launchers from files written by the Python test: node tests/js/run_serve.js <dir>
// <dir>/spec.json: {T, B, nHq, nKv, hd, page, pages, width, P, K, N, r, n, V, top, files: [names of raw files]}; results as <name>.out
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
const { T, B, nHq, nKv, hd, page, pages, width, P, K, N, r, n, V, top } = s;

const rows = page * pages * nKv;
const pool = { kq: zeros(rows * hd), ks: zeros(rows * hd / 8), vq: zeros(rows * hd), vs: zeros(rows * hd / 8), page, pages };
const table = { buf: b.table, width, B };
const qr = zeros(T * nHq * hd * 4), o = zeros(B * nHq * hd * 4);
const ld = (nHq + 2 * nKv) * hd, k = E.view(b.qkv, nHq * hd * 4), v = E.view(b.qkv, (nHq + nKv) * hd * 4);
L.attnPrepPagedQ8(b.qkv, k, v, b.qw, b.kw, qr, pool, table, b.seq, b.pos, b.rot, T, nHq, nKv, hd, 1e6, 1e-6, ld, ld);
save('qr', qr, T * nHq * hd * 4);
save('kq', pool.kq, rows * hd);
save('ks', pool.ks, rows * hd / 8);
save('vq', pool.vq, rows * hd);
L.attnSharedQ8(qr, pool, table, b.lens, { starts: b.starts, shared: b.shared, P }, o, nHq, nKv, hd);
save('o', o, B * nHq * hd * 4);
// without norms and q, with the positions for the rotation: what a cache of keys needs
L.attnPrepPagedQ8(null, k, v, null, null, null, pool, table, b.seq, b.pos, null, T, 0, nKv, hd, 1e6, 1e-6, ld, ld);
save('kq2', pool.kq, rows * hd);

L.loraAdd(b.x, b.idx, { a: b.a, b: b.b, scale: b.scale, n, r, K, N, bf16: false }, b.y, B);
save('y', b.y, B * N * 4);
const lp = { lp: zeros(B * 4), entropy: zeros(B * 4), rank: zeros(B * 4), topIds: zeros(B * top * 4), topLp: zeros(B * top * 4) };
L.logprobs(b.logits, b.ids, lp, B, V, top);
for (const f of Object.keys(lp)) save(f, lp[f], B * (f.startsWith('top') ? top : 1) * 4);
const only = zeros(B * 4);
L.logprobs(b.logits, b.ids, { lp: only }, B, V);
save('only', only, B * 4);
let refused = '';
try { L.logprobs(b.logits, b.ids, { lp: only }, B, V, V + 1); } catch (e) { refused = e.message; }
fs.writeFileSync(path.join(dir, 'refused.out'), refused);
process.exit(0);
