"""The shim's draft-tree methods (draftTree, encodeLayerTree, acceptTree, keepRows) through the Node-API addon: run by tests/js/tree_case.js, whose outputs are checked here against the 64-bit oracle
with the roundings' bound of the C ABI's own tests; the addon's table of those calls."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest
from oracle import attn_oracle as O
from oracle import tree_oracle as T
from pooled_amd.capi import tree_of_parents

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_addon_exports_when_built():
    addon = os.path.join(ROOT, "pooled_amd", "lib", "pooled_attn.node")
    if not (os.path.exists(addon) and shutil.which("node")):
        pytest.skip("addon or node missing")
    js = "const a=require(%r); for (const w of ['setRopeAxes','glueKvAt','attnTree','kvCompact']) { let ok = 0; try { a[w](); } catch (e) { ok = e instanceof TypeError; } if (!ok) throw new Error(w); } console.log('ok');" % addon
    r = subprocess.run(["node", "-e", js], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.mark.gpu
@pytest.mark.skipif(shutil.which("node") is None, reason="node not installed")
@pytest.mark.parametrize("q8", [False, True])
def test_a_tree_through_the_shim(tmp_path, q8):
    cfg = dict(n_heads=4, n_kv_heads=2, head_dim=256, n_rot=64, rope_theta=1e6, eps=1e-6, qk_norm=True, gate=True)
    base, parents, leaf = 90, [-1, 0, 0, 1, 2, 4, -1, 6, 5, 5, 8], 10
    seen, n = tree_of_parents(parents), len(parents)
    path = [int(c) for c in np.nonzero(seen[leaf])[0]]
    d = O.make_inputs(cfg, 0, base + n + 1, 7)
    for name, arr in (("q", d["qraw"]), ("k", d["kraw"]), ("v", d["vraw"]), ("qw", d["qw"]), ("kw", d["kw"])):
        np.ascontiguousarray(arr, np.float32).tofile(tmp_path / (name + ".bin"))
    (tmp_path / "case.json").write_text(json.dumps(dict(nH=4, nKV=2, hd=256, nRot=64, maxSeq=128, cols=90, base=base, parents=parents, leaf=leaf, path=path, q8=q8)))
    r = subprocess.run(["node", os.path.join(ROOT, "tests", "js", "tree_case.js"), str(tmp_path)], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr)
    assert r.returncode == 0 and "TREE DONE" in r.stdout, r.stdout + r.stderr
    get = lambda name, t: np.fromfile(tmp_path / (name + ".out"), t).reshape(base + n, 2, -1)  # noqa: E731
    k, v = (O.q8_dequantize(get("kv%d" % t, np.int8), get("kv%d" % (t + 2), np.float32)) if q8 else get("kv%d" % t, np.float16).astype(np.float32) for t in range(2))
    rows = slice(base, base + n)
    pre = T.glue_at(d["qraw"][rows], d["kraw"][rows], d["vraw"][rows], d["qw"], d["kw"], (base + seen.sum(1) - 1)[None], np.zeros(32, int), cfg)
    ref, absolute, reach = T.tree_attention(pre["q"], k, v, base, seen, pre["gate"])
    got = np.fromfile(tmp_path / "out.out", np.float32).reshape(ref.shape)
    off, bound = np.abs(got - ref), T.tree_bound(ref, absolute, reach, np.abs(v).max(), base + n, q8)
    print("tree through the shim: max-abs %.2e, %.1f %% of the bound" % (off.max(), 100 * (off / bound).max()))
    assert (off <= bound).all()
