"""No-GPU check of what the shim's draftTree refuses and sends, over an addon whose calls are recorded instead of made."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ADDON = os.path.join(ROOT, "pooled_amd", "lib", "pooled_attn.node")

PROGRAM = r"""
const { HipAttention, addon } = require(process.argv[1]);
let sent = [];
addon.malloc = (ctx, bytes) => bytes; addon.upload = (ctx, ptr, a) => { sent.push(Array.from(a)); };
addon.deltaCreate = () => { throw new Error("deltaCreate reached"); };
const make = (more) => Object.assign(Object.create(HipAttention.prototype), { ctx: 0, NC: 6, maxSeq: 100, verifyExact: false }, more);
const refused = (e, parents, base, pos0, what) => {
  sent = [];
  let text = "";
  try { e.draftTree(parents, base, pos0); } catch (x) { text = x.message; }
  if (text.indexOf("draftTree: ") !== 0 || text.indexOf(what) < 0 || sent.length) throw new Error("not refused: " + what + " (" + text + ")");
};
const e = make({});
for (const base of [-1, 95, 2.5, "7", undefined, NaN]) refused(e, [-1, 0, 0, 1, 2, 3], base, 0, "maxSeq");
for (const pos0 of [-1, 0.5, 4294967291, null, NaN]) refused(e, [-1, 0, 0, 1, 2, 3], 90, pos0, "pos0");
refused(e, [], 0, 0, "0 columns");
refused(e, [0], 0, 0, "parent");
refused(make({ verifyExact: true }), [-1], 0, 0, "verifyExact");
const hybrid = make({ delta: {} });
for (const parents of [[-1, 0, 0], [-1, -1], [-1, 0, 1, 0]]) refused(hybrid, parents, 5, 5, "chain");
sent = [];
hybrid.draftTree([-1, 0, 1], 5);                              // a chain goes through
if (JSON.stringify(sent[0]) !== "[1,3,7]" || JSON.stringify(sent[1].slice(0, 6)) !== "[5,6,7,0,0,0]") throw new Error(JSON.stringify(sent));
sent = [];
e.draftTree([-1, 0, 0, 2, -1, 4], 94, 4294967290);
if (JSON.stringify(sent[0]) !== "[1,3,5,13,16,48]" || JSON.stringify(sent[1].slice(18)) !== "[4294967290,4294967291,4294967291,4294967292,4294967290,4294967291]") throw new Error(JSON.stringify(sent));
let text = "";
try { e.initDelta({}); } catch (x) { text = x.message; }
if (text.indexOf("initDelta: a tree") !== 0) throw new Error("initDelta under a tree that branches: " + text);
refused(e, [-1, 9], 0, 0, "parent");                          // and the tree from before is still there
if (e._tree.n !== 6) throw new Error("a refused tree took the place of the one before");
console.log("ok");
"""


@pytest.mark.skipif(not os.path.exists(ADDON) or shutil.which("node") is None, reason="addon or node missing")
def test_trees_that_are_refused_and_sent():
    r = subprocess.run(["node", "-e", PROGRAM, os.path.join(ROOT, "pooled_amd", "js", "hip_attention.js")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
