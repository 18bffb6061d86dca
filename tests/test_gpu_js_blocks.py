"""The shim's delta-rule and experts methods (initDelta, encodeDelta, upMoe, encodeMoe) through the Node-API addon: a prompt, a draft of which some columns are accepted, a
token, then a layer of experts, run by tests/js/blocks_case.js and checked here against the 64-bit oracle, with the tolerances of the C ABI's own tests."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest
from oracle import blocks_oracle as B
from pooled_amd.capi import PA_W_Q8_0
from test_gpu_delta import step_tol
from test_gpu_moe import close as moe_close, experts

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("node") is None, reason="node not installed")
def test_blocks_through_the_shim(tmp_path):
    rng = np.random.default_rng(8)
    nk, nv, hk, hv, w, n, draft, accepted = 2, 4, 64, 32, 4, 70, 5, 3
    total, ch = n + draft, 2 * nk * hk + nv * hv
    dim, ffn, E, top, cols = 256, 96, 12, 3, 6
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    qkv, a, b, conv, bias, a_log, dt = f(total, ch), f(total, nv), f(total, nv), f(ch, w) / 2, 0.1 * f(ch), f(nv), f(nv)
    ex, sh = experts(rng, PA_W_Q8_0, E, dim, ffn), dict(experts(rng, PA_W_Q8_0, 0, dim, ffn), weight=f(dim) / 16)
    router, norm, x = 1.5 * f(E, dim) / 16, 1 + 0.1 * f(dim), 2 * f(cols, dim)
    files = dict(qkv=qkv, a=a, b=b, conv=conv, bias=bias, a_log=a_log, dt=dt, router=router, norm=norm, x=x, sharedGate=sh["weight"])
    for k, js in (("gate", "Gate"), ("up", "Up"), ("down", "Down")):
        files.update({k: ex[k], k + "Scales": ex[k + "_s"], "shared%sW" % js: sh[k], "shared%sScales" % js: sh[k + "_s"]})
    for name, arr in files.items():
        np.ascontiguousarray(arr).tofile(tmp_path / (name + ".bin"))
    (tmp_path / "case.json").write_text(json.dumps(dict(nk=nk, nv=nv, hk=hk, hv=hv, w=w, n=n, draft=draft, accepted=accepted,
                                                        moe=dict(dim=dim, ffn=ffn, experts=E, top=top, n=cols))))
    r = subprocess.run(["node", os.path.join(ROOT, "tests", "js", "blocks_case.js"), str(tmp_path)], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr)
    assert r.returncode == 0 and "BLOCKS DONE" in r.stdout, r.stdout + r.stderr
    get = lambda name: np.fromfile(tmp_path / (name + ".out"), np.float32)  # noqa: E731

    def oracle(order):
        c, g, beta, st = B.delta_glue(qkv[order], conv, bias, a[order], b[order], a_log, dt, np.zeros((w - 1, ch)))
        m, key = len(order), nk * hk
        o, S = B.delta_rule(c[:, :key].reshape(m, nk, hk), c[:, key:2 * key].reshape(m, nk, hk), c[:, 2 * key:].reshape(m, nv, hv), g, beta, np.zeros((nv, hv, hk)))
        return o, S, st
    whole, _, _ = oracle(list(range(total)))
    line = list(range(n + accepted)) + [n + accepted]
    tail, S, st = oracle(line)
    ref = np.concatenate([whole, tail[-1:]])
    got = get("delta").reshape(ref.shape).astype(np.float64)
    # the rule's own bound, and the pre-step's 12 roundings, which it passes on as it does those of its inputs; a head's norm over all columns
    bound = 8 * step_tol(total) + 4 * 12 * 2.0 ** -24 * (1 + total ** 0.5)
    d = np.sqrt(((got - ref) ** 2).sum((0, 2)) / (ref ** 2).sum((0, 2)))
    print("delta %.2e of %.2e" % (d.max(), bound))
    assert np.all(d <= bound)
    s = get("state").reshape(S.shape)
    assert np.all(np.sqrt(((s - S) ** 2).sum((1, 2)) / (S ** 2).sum((1, 2))) <= bound)
    assert np.array_equal(get("inputs").reshape(st.shape), st.astype(np.float32))
    y, _, _ = B.moe_layer(x, norm, router, ex, top, PA_W_Q8_0, True, sh)
    moe_close(get("y").reshape(y.shape), x, y, "experts")
