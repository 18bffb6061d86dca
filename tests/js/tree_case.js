// usage: node tree_case.js DIR -- the shim's draft-tree methods over the inputs in DIR; writes what they give beside them, for the caller to check
"use strict";
const fs = require("fs"), path = require("path");
const { HipAttention } = require(path.join(__dirname, "..", "..", "pooled_amd", "js", "hip_attention.js"));
const dir = process.argv[2];
const C = JSON.parse(fs.readFileSync(path.join(dir, "case.json"), "utf8"));
const f32 = (n) => { const b = fs.readFileSync(path.join(dir, n + ".bin")); return new Float32Array(b.buffer.slice(b.byteOffset, b.byteOffset + b.length)); };
const save = (n, a) => fs.writeFileSync(path.join(dir, n + ".out"), Buffer.from(a.buffer, a.byteOffset, a.byteLength));
const throws = (f, what) => { try { f(); } catch (e) { return; } throw new Error("not refused: " + what); };
const same = (a, b) => Buffer.from(a.buffer, a.byteOffset, a.byteLength).equals(Buffer.from(b.buffer, b.byteOffset, b.byteLength));

const make = () => {
  const e = new HipAttention({ nH: C.nH, nKV: C.nKV, hd: C.hd, nRot: C.nRot, ropeTheta: 1e6, eps: 1e-6, maxSeq: C.maxSeq, nLayers: 2, batchCols: C.cols, gate: true, kvQ8: C.q8 });
  for (let i = 0; i < 2; i++) e.setLayerNorms(i, f32("qw"), f32("kw"));
  return e;
};
const q = f32("q"), k = f32("k"), v = f32("v");
const load = (e, rows) => rows.forEach((r, c) => {
  e.writeColumn(e.B.qFull, c, q.subarray(r * e.B.qFull.n, (r + 1) * e.B.qFull.n));
  e.writeColumn(e.B.k, c, k.subarray(r * e.B.k.n, (r + 1) * e.B.k.n));
  e.writeColumn(e.B.v, c, v.subarray(r * e.B.v.n, (r + 1) * e.B.v.n));
});
const range = (a, n) => Array.from({ length: n }, (_, i) => a + i);
const a = make(), b = make(), n = C.parents.length;
for (const e of [a, b]) { load(e, range(0, C.base)); for (let i = 0; i < 2; i++) e.encodeGlueDense(null, i, 0, C.base); }

throws(() => a.encodeLayerTree(null, 0), "no tree");
throws(() => a.draftTree([0], C.base), "a column that is its own parent");
throws(() => a.draftTree(new Array(C.cols + 1).fill(-1), C.base), "more columns than batchCols");
throws(() => a.setRopeAxes([0, 1]), "short list of axes");
throws(() => a.setRopeAxes(new Array(C.nRot / 2).fill(4)), "a fifth axis");
throws(() => a.keepRows(5, [4]), "a row in front of dstRow");
throws(() => a.keepRows(5, [7, 7]), "the same row twice");
a.setRopeAxes(range(0, C.nRot / 2).map((i) => i % 3));            // the same position on every axis: what one axis gives
a.draftTree(C.parents, C.base);
load(a, range(C.base, n));
for (let i = 0; i < 2; i++) a.encodeLayerTree(null, i);
a.sync();
const outs = a.readAttnOut(n), all = new Float32Array(n * C.nH * C.hd);
outs.forEach((o, i) => all.set(o, i * C.nH * C.hd));
save("out", all);
for (let t = 0; t < (C.q8 ? 4 : 2); t++) save("kv" + t, a.kvRead(1, t, 0, C.base + n));
throws(() => a.acceptTree(n), "no such column");
const kept = a.acceptTree(C.leaf);
if (JSON.stringify(kept) !== JSON.stringify(C.path)) throw new Error("path " + kept);
throws(() => a.acceptTree(0), "a tree that was accepted before");
load(b, kept.map((c) => C.base + c));                             // the same tokens one behind the other
for (let i = 0; i < 2; i++) b.encodeGlueDense(null, i, C.base, kept.length);
for (let i = 0; i < 2; i++) for (let t = 0; t < (C.q8 ? 4 : 2); t++)
  if (!same(a.kvRead(i, t, 0, C.base + kept.length), b.kvRead(i, t, 0, C.base + kept.length))) throw new Error("cache " + t + " of layer " + i);
for (const e of [a, b]) { load(e, [C.base + n]); e.encodeLayerAttn(null, 1, C.base + kept.length); e.sync(); }
if (!same(a.readColumn(a.B.attnOut, 0), b.readColumn(b.B.attnOut, 0))) throw new Error("the next token");
const rows = range(0, C.base).filter((r) => r % 3 !== 1).filter((r) => r >= 10), before = a.kvRead(0, 1, 0, C.base);
a.keepRows(10, rows);
const per = before.length / C.base, after = a.kvRead(0, 1, 0, C.base);
rows.forEach((r, i) => { if (!same(after.subarray((10 + i) * per, (11 + i) * per), before.subarray(r * per, (r + 1) * per))) throw new Error("keepRows: row " + i); });
a.destroy(); b.destroy();
console.log("TREE DONE");
