"""Columns at rotary positions of their own through the shim (setRopeAxes, setPositions, encodeLayerAt) on the GPU: a prompt with an image in two chunks and two tokens behind it, run by
tests/js/positions_case.js.  The cache rows are the oracle's, bit for bit; the outputs are within the path's tolerance of causal attention over them."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest
from oracle import attn_oracle as O
from oracle import tree_oracle as T
from helpers import MAX_ABS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
@pytest.mark.skipif(shutil.which("node") is None, reason="node not installed")
@pytest.mark.parametrize("q8", [False, True])
def test_a_prompt_with_an_image(tmp_path, q8):
    cfg = dict(n_heads=4, n_kv_heads=2, head_dim=256, n_rot=64, rope_theta=1e6, eps=1e-6, qk_norm=True, gate=True)
    chunks, rows = [40, 33, 1, 1], 75
    # ten words, an image of 6 x 10 patches at one time, words behind it that go on from its longer side
    c = np.arange(60)
    pos = np.concatenate([np.stack([np.arange(10)] * 3), np.stack([0 * c + 10, c // 10 + 10, c % 10 + 10]), np.stack([np.arange(5) + 20] * 3)], 1)
    assert pos.shape == (3, rows)
    axis = np.arange(32) % 3
    d = O.make_inputs(cfg, 0, rows, 11)
    for name, arr in (("q", d["qraw"]), ("k", d["kraw"]), ("v", d["vraw"]), ("qw", d["qw"]), ("kw", d["kw"])):
        np.ascontiguousarray(arr, np.float32).tofile(tmp_path / (name + ".bin"))
    (tmp_path / "case.json").write_text(json.dumps(dict(nH=4, nKV=2, hd=256, nRot=64, maxSeq=128, cols=40, rows=rows, chunks=chunks, axis=axis.tolist(), positions=pos.tolist(), q8=q8)))
    r = subprocess.run(["node", os.path.join(ROOT, "tests", "js", "positions_case.js"), str(tmp_path)], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr)
    assert r.returncode == 0 and "POSITIONS DONE" in r.stdout, r.stdout + r.stderr
    pre = T.glue_at(d["qraw"], d["kraw"], d["vraw"], d["qw"], d["kw"], pos, axis, cfg)
    line = T.glue_at(d["qraw"], d["kraw"], d["vraw"], d["qw"], d["kw"], np.stack([np.arange(rows)] * 3), axis, cfg)
    assert np.abs(pre["k"] - line["k"]).max() > 0.5                                   # rows turned by their numbers would be others
    want = [*O.q8_quantize(pre["k"])[:1], *O.q8_quantize(pre["v"])[:1], O.q8_quantize(pre["k"])[1], O.q8_quantize(pre["v"])[1]] if q8 else [O.f16_bits(pre["k"]), O.f16_bits(pre["v"])]
    for t, w in enumerate(want):
        got = np.fromfile(tmp_path / ("kv%d.out" % t), w.dtype).reshape(w.shape)
        assert np.array_equal(got, w), t
    k, v = (O.q8_dequantize(want[t], want[t + 2]) if q8 else O.f16_round(pre["kv"[t]]) for t in range(2))
    ref = T.tree_attention(pre["q"], k, v, 0, np.tril(np.ones((rows, rows), bool)), pre["gate"])[0]
    got = np.fromfile(tmp_path / "out.out", np.float32).reshape(ref.shape)
    print("image prompt: max-abs %.2e of %.2f" % (np.abs(got - ref).max(), np.abs(ref).max()))
    assert np.abs(got - ref).max() <= MAX_ABS
