// usage: node blocks_case.js DIR -- the shim's delta-rule and experts methods over the inputs in DIR; writes what they give beside them, for the caller to check
"use strict";
const fs = require("fs"), path = require("path");
const { HipAttention, addon } = require(path.join(__dirname, "..", "..", "pooled_amd", "js", "hip_attention.js"));
const dir = process.argv[2];
const C = JSON.parse(fs.readFileSync(path.join(dir, "case.json"), "utf8"));
const bytes = (n) => fs.readFileSync(path.join(dir, n + ".bin"));
const raw = (n, T) => { const b = bytes(n); return new T(b.buffer.slice(b.byteOffset, b.byteOffset + b.length)); };
const f32 = (n) => raw(n, Float32Array);
const save = (n, a) => fs.writeFileSync(path.join(dir, n + ".out"), Buffer.from(a.buffer, a.byteOffset, a.byteLength));
const throws = (f, what) => { try { f(); } catch (e) { return; } throw new Error("not refused: " + what); };

const eng = new HipAttention({ nH: 1, nKV: 1, hd: 128, ropeTheta: 1e6, eps: 1e-6, maxSeq: 64, nLayers: 1, batchCols: C.n });
throws(() => eng.initDelta({ nKHeads: 3, nVHeads: 4, headK: 64, headV: 32, convWidth: 4 }), "nVHeads not a multiple");
eng.initDelta({ nKHeads: C.nk, nVHeads: C.nv, headK: C.hk, headV: C.hv, convWidth: C.w, nLayers: 2 });
throws(() => eng.encodeDelta(null, 1, 1), "layer without weights");
throws(() => eng.setDeltaLayer(1, { convW: new Float32Array(3), convB: null, aLog: new Float32Array(C.nv), dtBias: new Float32Array(C.nv) }), "short convW");
eng.setDeltaLayer(1, { convW: f32("conv"), convB: f32("bias"), aLog: f32("a_log"), dtBias: f32("dt") });
const qkv = f32("qkv"), a = f32("a"), b = f32("b"), ch = eng.delta.channels;
const load = (from, n) => { for (let c = 0; c < n; c++) {
  eng.writeColumn(eng.B.dQkv, c, qkv.subarray((from + c) * ch, (from + c + 1) * ch));
  eng.writeColumn(eng.B.dA, c, a.subarray((from + c) * C.nv, (from + c + 1) * C.nv));
  eng.writeColumn(eng.B.dB, c, b.subarray((from + c) * C.nv, (from + c + 1) * C.nv));
} };
const out = [];
const keep = (n) => { for (let c = 0; c < n; c++) out.push(eng.readColumn(eng.B.dOut, c)); };
load(0, C.n); eng.encodeDelta(null, 1, C.n); eng.sync(); keep(C.n);                             // the prompt
const before = eng.readDelta(1);
load(C.n, C.draft); eng.encodeDelta(null, 1, C.draft, { commit: 0 }); eng.sync(); keep(C.draft);   // a draft ...
const draft = eng.readDelta(1);
if (!Buffer.from(before.S.buffer).equals(Buffer.from(draft.S.buffer)) || !Buffer.from(before.conv.buffer).equals(Buffer.from(draft.conv.buffer))) throw new Error("a draft moved the state");
eng.encodeDelta(null, 1, C.accepted, { stateOnly: true });                                      // ... of which so many columns are accepted
load(C.n + C.accepted, 1); eng.encodeDelta(null, 1, 1); eng.sync(); keep(1);                    // and a token
const all = new Float32Array(out.length * C.nv * C.hv);
out.forEach((o, i) => all.set(o, i * C.nv * C.hv));
save("delta", all);
const st = eng.readDelta(1);
save("state", st.S); save("inputs", st.conv);
eng.resetDelta();
if (eng.readDelta(1).S.some((v) => v !== 0)) throw new Error("resetDelta");
eng.writeDelta(0, st);
if (!Buffer.from(eng.readDelta(0).S.buffer).equals(Buffer.from(st.S.buffer))) throw new Error("writeDelta");
throws(() => eng.writeDelta(0, { S: new Float32Array(5), conv: st.conv }), "short state");

const M = C.moe, planes = { router: f32("router"), sharedGate: f32("sharedGate") };
for (const k of ["gate", "up", "down", "sharedGateW", "sharedUpW", "sharedDownW"]) planes[k] = raw(k, Int8Array);
for (const k of ["gateScales", "upScales", "downScales", "sharedGateScales", "sharedUpScales", "sharedDownScales"]) planes[k] = raw(k, Uint16Array);
throws(() => eng.upMoe({ kind: "q8", dim: M.dim, ffn: M.ffn, nExperts: M.experts + 1, topK: M.top, normTopk: true, planes: planes }), "short planes");
throws(() => eng.upMoe({ kind: "q8", dim: M.dim, ffn: M.ffn, nExperts: M.experts, topK: M.experts + 1, normTopk: true, planes: planes }), "topK");
const moe = eng.upMoe({ kind: "q8", dim: M.dim, ffn: M.ffn, nExperts: M.experts, topK: M.top, normTopk: true, planes: planes });
const nw = addon.malloc(eng.ctx, M.dim * 4);
addon.upload(eng.ctx, nw, f32("norm"));
const X = eng.residualCols(M.dim), x = f32("x");
for (let c = 0; c < M.n; c++) eng.writeColumn(X, c, x.subarray(c * M.dim, (c + 1) * M.dim));
eng.encodeMoe(null, moe, nw, X, M.n);
eng.sync();
const y = new Float32Array(M.n * M.dim);
for (let c = 0; c < M.n; c++) y.set(eng.readColumn(X, c), c * M.dim);
save("y", y);
addon.free(eng.ctx, nw);
eng.destroy();
console.log("BLOCKS DONE");
