"""The pre-step of columns with positions of their own (pa_glue_kv_at) on the GPU: q, gate and cache rows against the oracle, bit for bit, and
against pa_glue_kv where the positions are base + c."""
import numpy as np
import pytest
from oracle import attn_oracle as O
from oracle import tree_oracle as T
from pooled_amd.capi import PooledAttn, PA_ERR_INVALID
from helpers import SHAPES

pytestmark = pytest.mark.gpu


class Inputs:
    def __init__(self, pa, d, gap=0):
        pad = lambda a: np.concatenate([a, np.full((a.shape[0], gap), np.nan, np.float32)], 1) if gap else a  # noqa: E731
        self.q, self.k, self.v = (pa.to_device(pad(d[x])) for x in ("qraw", "kraw", "vraw"))
        self.strides = [d[x].shape[1] + gap for x in ("qraw", "kraw", "vraw")]
        self.qw, self.kw = pa.to_device(d["qw"]), pa.to_device(d["kw"])

    def call(self, pa, layer, pos, row, n, stride=None):
        p = pa.to_device(np.ascontiguousarray(pos, np.uint32))
        pa.glue_kv_at(layer, self.q, self.strides[0], self.k, self.strides[1], self.v, self.strides[2], self.qw, self.kw, p, pos.shape[1] if stride is None else stride, row, n)
        pa.sync()


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32 if a.dtype == np.float32 else a.dtype)


def axes_of(kind, half):
    i = np.arange(half)
    return {"one": i * 0, "turns": i % 3, "ranges": np.minimum(i * 3 // half, 2), "four": i % 4, "two": (i < half // 3).astype(int)}[kind]


@pytest.mark.parametrize("kind", ["one", "two", "turns", "ranges", "four"])
@pytest.mark.parametrize("shape", sorted(SHAPES) + ["plain"])
@pytest.mark.parametrize("n,row,gap", [(1, 0, 0), (5, 7, 64), (17, 100, 0), (70, 3, 4)])
def test_positions_of_any_axes(shape, kind, n, row, gap):
    cfg = dict(SHAPES.get(shape) or dict(SHAPES["qwen3_1p7b"], qk_norm=False, n_rot=96, n_heads=6, n_kv_heads=3))
    half, seq = cfg["n_rot"] // 2, row + n + 5
    rng = np.random.default_rng(n + row)
    d = O.make_inputs(cfg, 0, n, n)
    axis = axes_of(kind, half)
    pos = rng.integers(0, seq, (axis.max() + 1, n + 3))                   # three positions behind the call's
    pos[:, n // 2] = seq + 100000                                          # behind the table
    ref = T.glue_at(d["qraw"], d["kraw"], d["vraw"], d["qw"], d["kw"], pos[:, :n], axis, cfg)
    with PooledAttn(cfg, seq, n_layers=2, max_cols=n) as pa:
        pa.layer_alloc(1)
        pattern = (np.arange(seq * cfg["n_kv_heads"] * cfg["head_dim"], dtype=np.uint32) * 40503 >> 3).astype(np.uint16).reshape(seq, cfg["n_kv_heads"], cfg["head_dim"])
        pa.kv_write(1, 0, 0, pattern); pa.kv_write(1, 1, 0, pattern ^ 0x1111)
        if kind != "one":
            pa.set_rope_axes(axis)
        Inputs(pa, d, gap).call(pa, 1, pos, row, n)
        assert np.array_equal(bits(pa.read_q_buffer(n)), bits(ref["q"]))
        if cfg["gate"]:
            assert np.array_equal(bits(pa.read_gate_buffer(n)), bits(ref["gate"]))
        K, V = pa.kv_read(1, 0, 0, seq), pa.kv_read(1, 1, 0, seq)
    pattern_v = pattern ^ 0x1111
    pattern[row:row + n], pattern_v[row:row + n] = O.f16_bits(ref["k"]), O.f16_bits(ref["v"])
    assert np.array_equal(K, pattern) and np.array_equal(V, pattern_v)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_positions_in_a_line_are_glue_kv(shape, q8):
    """base + c on one axis, and on three: q, gate and every cache tensor have pa_glue_kv's bits."""
    cfg = dict(SHAPES[shape], kv_q8=q8)
    for n, base in ((1, 0), (37, 901)):
        d = O.make_inputs(cfg, 0, n, base + 5)
        line = base + np.arange(n)
        with PooledAttn(cfg, base + n, n_layers=3, max_cols=n) as pa:
            for l in range(3):
                pa.layer_alloc(l)
            seen = []
            tensors = range(4 if q8 else 2)

            def keep(l):
                seen.append([bits(pa.read_q_buffer(n))] + ([bits(pa.read_gate_buffer(n))] if cfg["gate"] else []) + [bits(pa.kv_read(l, w, 0, base + n)) for w in tensors])
            pa.run_glue_kv(0, d["qraw"], d["kraw"], d["vraw"], d["qw"], d["kw"], base)
            keep(0)
            x = Inputs(pa, d)
            x.call(pa, 1, line[None], base, n, stride=0)
            keep(1)
            pa.set_rope_axes(np.arange(cfg["n_rot"] // 2) % 3)
            x.call(pa, 2, np.stack([line] * 3), base, n)
            keep(2)
        for other in seen[1:]:
            assert len(other) == len(seen[0]) and all(np.array_equal(a, b) for a, b in zip(seen[0], other))


def test_int8_rows_of_turned_columns():
    """Int8 values and scales are those of the oracle's quantisation of the turned rows."""
    cfg = dict(SHAPES["qwen38_27b"], kv_q8=True)
    n, row = 9, 33
    d = O.make_inputs(cfg, 0, n, 3)
    axis = axes_of("ranges", cfg["n_rot"] // 2)
    pos = np.random.default_rng(0).integers(0, 60, (3, n))
    ref = T.glue_at(d["qraw"], d["kraw"], d["vraw"], d["qw"], d["kw"], pos, axis, cfg)
    with PooledAttn(cfg, 64, n_layers=1, max_cols=n) as pa:
        pa.layer_alloc(0)
        pa.set_rope_axes(axis)
        Inputs(pa, d).call(pa, 0, pos, row, n)
        for w, x in ((0, ref["k"]), (1, ref["v"])):
            val, sc = O.q8_quantize(x)
            assert np.array_equal(pa.kv_read(0, w, row, n), val) and np.array_equal(bits(pa.kv_read(0, w + 2, row, n)), bits(sc))
            assert not pa.kv_read(0, w, 0, row).any() and not pa.kv_read(0, w, row + n, 64 - row - n).any()


@pytest.mark.parametrize("far", [1 << 20, (1 << 24) + 1, 0x7FFFFFFF, 0xFFFFFFFF])
def test_far_positions(far):
    """Positions behind the table, up to the largest: the angle is the f32 product, its cosine and sine exact to f32."""
    cfg = SHAPES["qwen36_moe"]
    d = O.make_inputs(cfg, 0, 3, 1)
    pos = np.array([[far, 5, far - 1]])
    ref = T.glue_at(d["qraw"], d["kraw"], d["vraw"], d["qw"], d["kw"], pos, axes_of("one", 32), cfg)
    with PooledAttn(cfg, 16, n_layers=1, max_cols=3) as pa:
        pa.layer_alloc(0)
        Inputs(pa, d).call(pa, 0, pos, 2, 3)
        assert np.array_equal(bits(pa.read_q_buffer(3)), bits(ref["q"]))
        assert np.array_equal(pa.kv_read(0, 0, 2, 3), O.f16_bits(ref["k"]))


def test_many_columns():
    """A prompt chunk with an image: 700 columns, three axes."""
    cfg = SHAPES["qwen38_27b"]
    n, row = 700, 1234
    d = O.make_inputs(cfg, 0, n, 6)
    axis = axes_of("turns", 32)
    c = np.arange(n)
    pos = np.stack([c // 400 + 600, c // 20 % 20 + 600, c % 20 + 600])
    ref = T.glue_at(d["qraw"], d["kraw"], d["vraw"], d["qw"], d["kw"], pos, axis, cfg)
    with PooledAttn(cfg, row + n, n_layers=1, max_cols=n) as pa:
        pa.layer_alloc(0)
        pa.set_rope_axes(axis)
        Inputs(pa, d).call(pa, 0, pos, row, n)
        assert np.array_equal(bits(pa.read_q_buffer(n)), bits(ref["q"])) and np.array_equal(bits(pa.read_gate_buffer(n)), bits(ref["gate"]))
        assert np.array_equal(pa.kv_read(0, 0, row, n), O.f16_bits(ref["k"])) and np.array_equal(pa.kv_read(0, 1, row, n), O.f16_bits(ref["v"]))
        assert not pa.kv_read(0, 0, 0, row).any()


def test_refusals():
    cfg = SHAPES["qwen36_moe"]
    qc, kvd = cfg["n_heads"] * cfg["head_dim"] * 2, cfg["n_kv_heads"] * cfg["head_dim"]
    with PooledAttn(cfg, 100, n_layers=2, max_cols=8) as pa:
        pa.layer_alloc(0)
        q, k, v, w, pos = pa.alloc(8 * qc * 4), pa.alloc(8 * kvd * 4), pa.alloc(8 * kvd * 4), pa.alloc(1024), pa.alloc(256)
        good = dict(layer=0, q=q.ptr, qs=qc, k=k.ptr, ks=kvd, v=v.ptr, vs=kvd, qw=w.ptr, kw=w.ptr, pos=pos.ptr, ps=8, row=92, n=8)

        def call(**change):
            a = dict(good, **change)
            return pa.L.pa_glue_kv_at(pa.ctx, a["layer"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["qw"], a["kw"], a["pos"], a["ps"], a["row"], a["n"])
        for change in (dict(layer=1), dict(layer=9), dict(n=0), dict(n=9), dict(row=93), dict(row=0xFFFFFFFF), dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(qw=None), dict(kw=None),
                       dict(qs=qc - 1), dict(ks=kvd - 1), dict(vs=kvd - 1), dict(pos=pos.ptr + 2), dict(q=q.ptr + 1), dict(k=k.ptr + 2), dict(q=pa.q_buffer_ptr()), dict(v=pa.gate_buffer_ptr() + 64)):
            assert call(**change) == PA_ERR_INVALID, change
            assert b"pa_glue_kv_at: " in pa.L.pa_last_error(pa.ctx), change
        half = cfg["n_rot"] // 2
        bad = np.zeros(half, np.uint8)
        bad[-1] = 2
        for n_axes, at in ((0, None), (5, None), (2, None), (2, bad.ctypes.data), (1, bad.ctypes.data)):
            assert pa.L.pa_set_rope_axes(pa.ctx, n_axes, at) == PA_ERR_INVALID
            assert b"pa_set_rope_axes: " in pa.L.pa_last_error(pa.ctx)
        with pytest.raises(ValueError):
            pa.set_rope_axes([0, 1])
        assert call(ps=0) == 0                       # one axis: its stride is not looked at
        pa.set_rope_axes(np.arange(half) % 3)
        assert call(ps=7) == PA_ERR_INVALID
        pa.set_rope_axes(None)
        assert call(ps=7) == 0
        pa.sync()
