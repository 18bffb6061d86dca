"""No-GPU check of the shim's setRopeAxes, setPositions and encodeLayerAt, over an addon whose calls are recorded instead of made."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ADDON = os.path.join(ROOT, "pooled_amd", "lib", "pooled_attn.node")

PROGRAM = r"""
const { HipAttention, addon } = require(process.argv[1]);
const calls = [];
for (const k of ["setRopeAxes", "upload", "glueKvAt", "attn"]) addon[k] = (...a) => { calls.push([k].concat(a.slice(1).map((x) => x && x.length !== undefined ? Array.from(x) : x))); };
addon.malloc = () => 7000; addon.gateBuffer = () => 42;
const buf = (ptr, n) => ({ ptr: ptr, stride: n * 4, n: n });
const make = (NC) => Object.assign(Object.create(HipAttention.prototype), { ctx: 0, NC: NC, dims: { nRot: 8, qDim: 16, kvDim: 8 }, gate: true, attnPrefillTile: true, _snapNow: null, outDtype: 0,
  _ones: 9, layers: [{ qNorm: 1, kNorm: 2 }], B: { qFull: buf(100, 32), k: buf(200, 8), v: buf(300, 8), attnOut: buf(400, 16) } });
const want = (w) => { if (JSON.stringify(calls) !== JSON.stringify(w)) throw new Error(JSON.stringify(calls) + " instead of " + JSON.stringify(w)); calls.length = 0; };
const refused = (f, what) => { let ok = false; try { f(); } catch (e) { ok = true; } if (!ok) throw new Error("not refused: " + what); want([]); };
const e = make(4);
refused(() => e.encodeLayerAt(null, 0, 0), "no positions");
refused(() => e.setPositions([[1, 2, 3, 4, 5]]), "more columns than batchCols");
refused(() => e.setPositions([[]]), "no columns");
refused(() => e.setPositions([]), "no axes");
refused(() => e.setPositions([[1], [1]]), "two axes where there is one");
refused(() => e.setPositions([[1.5]]), "half a position");
refused(() => e.setPositions([[-1]]), "a position in front of the first");
refused(() => e.setPositions([[4294967296]]), "a position beyond 32 bits");
e.setPositions([[11, 12]]);                                   // one axis
want([["upload", 7000, [11, 12, 0, 0]]]);
e.encodeLayerAt(null, 0, 50);
want([["glueKvAt", 0, 100, 32, 200, 8, 300, 8, 1, 2, 7000, 4, 50, 2], ["attn", 0, 0, null, 0, 42, 16, 50, 2, 400, 16, 0]]);
e.setRopeAxes([0, 1, 2, 0]);                                  // three: positions of one axis are no longer there
want([["setRopeAxes", 3, [0, 1, 2, 0]]]);
refused(() => e.encodeLayerAt(null, 0, 50), "positions of other axes");
refused(() => e.setPositions([[1, 2], [3, 4]]), "an axis missing");
refused(() => e.setPositions([[1, 2], [3, 4], [5]]), "a column missing");
e.setPositions([[1, 2, 3, 4], [5, 6, 7, 8], Uint32Array.from([9, 10, 11, 12])]);
want([["upload", 7000, [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12]]]);
e.encodeLayerAt(null, 0, 60);                                 // a pass of full width: the prefill kernel
want([["glueKvAt", 0, 100, 32, 200, 8, 300, 8, 1, 2, 7000, 4, 60, 4], ["attn", 1, 0, null, 0, 42, 16, 60, 4, 400, 16, 0]]);
e.setRopeAxes(null);
want([["setRopeAxes", 1, null]]);
e.setPositions([[3]]);
want([["upload", 7000, [3, 0, 0, 0]]]);
console.log("ok");
"""


@pytest.mark.skipif(not os.path.exists(ADDON) or shutil.which("node") is None, reason="addon or node missing")
def test_positions_reach_the_calls():
    r = subprocess.run(["node", "-e", PROGRAM, os.path.join(ROOT, "pooled_amd", "js", "hip_attention.js")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
