// usage: node positions_case.js DIR -- a prompt with an image, through the shim's columns at positions of their own: two chunks, then two tokens; writes outputs and caches beside the inputs
"use strict";
const fs = require("fs"), path = require("path");
const { HipAttention } = require(path.join(__dirname, "..", "..", "pooled_amd", "js", "hip_attention.js"));
const dir = process.argv[2];
const C = JSON.parse(fs.readFileSync(path.join(dir, "case.json"), "utf8"));
const f32 = (n) => { const b = fs.readFileSync(path.join(dir, n + ".bin")); return new Float32Array(b.buffer.slice(b.byteOffset, b.byteOffset + b.length)); };
const save = (n, a) => fs.writeFileSync(path.join(dir, n + ".out"), Buffer.from(a.buffer, a.byteOffset, a.byteLength));
const e = new HipAttention({ nH: C.nH, nKV: C.nKV, hd: C.hd, nRot: C.nRot, ropeTheta: 1e6, eps: 1e-6, maxSeq: C.maxSeq, nLayers: 2, batchCols: C.cols, gate: true, kvQ8: C.q8 });
for (let i = 0; i < 2; i++) e.setLayerNorms(i, f32("qw"), f32("kw"));
const q = f32("q"), k = f32("k"), v = f32("v"), all = new Float32Array(C.rows * C.nH * C.hd);
e.setRopeAxes(C.axis);
for (let at = 0; at < C.rows;) {
  const n = C.chunks.shift();
  for (let c = 0; c < n; c++) {
    const r = at + c;
    e.writeColumn(e.B.qFull, c, q.subarray(r * e.B.qFull.n, (r + 1) * e.B.qFull.n));
    e.writeColumn(e.B.k, c, k.subarray(r * e.B.k.n, (r + 1) * e.B.k.n));
    e.writeColumn(e.B.v, c, v.subarray(r * e.B.v.n, (r + 1) * e.B.v.n));
  }
  e.setPositions(C.positions.map((a) => a.slice(at, at + n)));
  for (let i = 0; i < 2; i++) e.encodeLayerAt(null, i, at);
  e.sync();
  e.readAttnOut(n).forEach((o, c) => all.set(o, (at + c) * C.nH * C.hd));
  at += n;
}
save("out", all);
for (let t = 0; t < (C.q8 ? 4 : 2); t++) save("kv" + t, e.kvRead(1, t, 0, C.rows));
e.destroy();
console.log("POSITIONS DONE");
