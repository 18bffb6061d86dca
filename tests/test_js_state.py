"""No-GPU check of the shim's writeDelta, over an addon whose state calls are recorded instead of made."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ADDON = os.path.join(ROOT, "pooled_amd", "lib", "pooled_attn.node")

PROGRAM = r"""
const { HipAttention, addon } = require(process.argv[1]);
const wrote = [];
addon.deltaStateBytes = (h, which) => which === 0 ? 64 : h === 1 ? 48 : 0;
addon.deltaWrite = (ctx, h, layer, which, a) => { wrote.push([layer, which, a.length]); };
const write = (handle, st) => { wrote.length = 0; let threw = false; try { HipAttention.prototype.writeDelta.call({ ctx: 0, delta: { handle: handle } }, 2, st); } catch (e) { threw = true; } return JSON.stringify([threw, wrote]); };
const f = (n) => new Float32Array(n);
const want = (got, w) => { if (got !== JSON.stringify(w)) throw new Error(got + " instead of " + JSON.stringify(w)); };
want(write(1, { S: f(16), conv: f(12) }), [false, [[2, 0, 16], [2, 1, 12]]]);
want(write(2, { S: f(16), conv: f(0) }), [false, [[2, 0, 16]]]);             // a handle without a convolution
want(write(1, { S: f(16), conv: f(11) }), [true, []]);                       // nothing is written of a state that does not fit
want(write(1, { S: f(15), conv: f(12) }), [true, []]);
want(write(1, { S: f(16) }), [true, []]);
want(write(2, { S: f(16), conv: f(12) }), [true, []]);
console.log("ok");
"""


@pytest.mark.skipif(not os.path.exists(ADDON) or shutil.which("node") is None, reason="addon or node missing")
def test_a_saved_state_that_does_not_fit_is_not_written_in_part():
    r = subprocess.run(["node", "-e", PROGRAM, os.path.join(ROOT, "pooled_amd", "js", "hip_attention.js")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
