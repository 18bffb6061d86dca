"""Attention of a draft tree over the cache (pa_attn_tree) on the GPU, against the oracle in 64 bits.  Tolerance per output: tree_oracle.tree_bound, the roundings that the call makes."""
import numpy as np
import pytest
from oracle import attn_oracle as O
from oracle import tree_oracle as T
from pooled_amd.capi import PooledAttn, PaError, PA_ERR_INVALID, PA_OUT_F16, PA_OUT_F32, tree_mask, tree_of_parents
from helpers import SHAPES

pytestmark = pytest.mark.gpu
NAN16 = 0x7E00


def random_tree(n, rng, roots=0.2):
    return tree_of_parents([-1 if c == 0 or rng.random() < roots else int(rng.integers(max(0, c - 6), c)) for c in range(n)])


class Case:
    """A context of `base` rows, a draft of n behind it, and rows of NaN behind that."""

    def __init__(self, cfg, base, n, seed, peak=1.0, more=40):
        rng = np.random.default_rng(seed)
        self.cfg, self.base, self.n, self.rng = cfg, base, n, rng
        nH, nKV, hd, T_ = cfg["n_heads"], cfg["n_kv_heads"], cfg["head_dim"], base + n
        self.rows = T_ + more
        self.q = (peak * rng.standard_normal((n, nH, hd))).astype(np.float32)
        self.gate = rng.standard_normal((n, nH, hd), dtype=np.float32) if cfg["gate"] else None
        k, v = (rng.standard_normal((T_, nKV, hd), dtype=np.float32) for _ in range(2))
        if cfg.get("kv_q8"):
            self.parts = [*O.q8_quantize(k)[:1], *O.q8_quantize(v)[:1], O.q8_quantize(k)[1], O.q8_quantize(v)[1]]
            self.k, self.v = O.q8_dequantize(self.parts[0], self.parts[2]), O.q8_dequantize(self.parts[1], self.parts[3])
        else:
            self.parts = [O.f16_bits(k), O.f16_bits(v)]
            self.k, self.v = O.f16_round(k), O.f16_round(v)
        self.seen = random_tree(n, rng)

    def fill(self, pa, layer=0):
        pa.layer_alloc(layer)
        for w, part in enumerate(self.parts):
            pa.kv_write(layer, w, 0, part)
            stale = np.full((self.rows - part.shape[0],) + part.shape[1:], 93 if w < 2 and self.cfg.get("kv_q8") else NAN16 if w < 2 else np.nan, part.dtype)
            pa.kv_write(layer, w, part.shape[0], stale)

    def context(self, **more):
        return PooledAttn(self.cfg, self.rows, n_layers=1, max_cols=max(self.n, 2), **more)

    def check(self, got, f16=False, seen=None, what=""):
        seen = self.seen if seen is None else seen
        ref, absolute, reach = T.tree_attention(self.q, self.k, self.v, self.base, seen, self.gate)
        bound = T.tree_bound(ref, absolute, reach, np.abs(self.v).max(), self.base + self.n, bool(self.cfg.get("kv_q8")), f16)
        off = np.abs(got.astype(np.float64) - ref)
        worst = float((off / bound).max())
        print("tree %s base %d n %d: max-abs %.2e, %.1f %% of the bound" % (what, self.base, self.n, off.max(), 100 * worst), flush=True)
        assert np.isfinite(got).all() and worst <= 1.0
        return worst


CASES = [(0, 1), (0, 5), (1, 1), (3, 2), (20, 13), (31, 1), (31, 33), (32, 8), (33, 31), (63, 64), (200, 7), (511, 32), (1000, 24), (1025, 65), (2011, 17), (4097, 3), (777, 100)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("base,n", CASES)
def test_trees(shape, base, n, q8):
    cfg = dict(SHAPES[shape], kv_q8=q8)
    f16 = (base + n) % 2 == 0
    c = Case(cfg, base, n, seed=base * 7 + n, peak=1.0 + (n % 3))
    with c.context() as pa:
        c.fill(pa)
        c.check(pa.run_attn_tree(0, c.q, c.seen, base, gate=c.gate, out_dtype=PA_OUT_F16 if f16 else PA_OUT_F32), f16, what=shape + (" q8" if q8 else ""))


@pytest.mark.parametrize("splits", [1, 2, 3, 5, 9, 16, 33, 64, 1000])
def test_any_number_of_splits(splits):
    for shape, base, n in (("qwen36_moe", 1000, 24), ("qwen3_1p7b", 1031, 9), ("qwen38_27b", 1050, 50)):
        c = Case(SHAPES[shape], base, n, seed=splits)
        with c.context() as pa:
            c.fill(pa)
            pa.set_decode_splits(splits)
            c.check(pa.run_attn_tree(0, c.q, c.seen, base, gate=c.gate), what="%s splits %d" % (shape, splits))


@pytest.mark.parametrize("heads,kv_heads,hd", [(1, 1, 128), (3, 3, 256), (7, 1, 128), (32, 1, 256), (64, 1, 128), (20, 4, 128)])
def test_head_layouts(heads, kv_heads, hd):
    cfg = dict(n_heads=heads, n_kv_heads=kv_heads, head_dim=hd, n_rot=64, rope_theta=1e6, eps=1e-6, qk_norm=True, gate=False)
    for q8 in (False, True):
        c = Case(dict(cfg, kv_q8=q8), 333, 11, seed=heads)
        with c.context() as pa:
            c.fill(pa)
            c.check(pa.run_attn_tree(0, c.q, c.seen, c.base), what="%d / %d heads of %d" % (heads, kv_heads, hd))


@pytest.mark.parametrize("base", [0, 77])
def test_masks_of_any_pattern(base):
    """Random bits, a column that sees every row, columns that see no drafted row: with no context in front those are zeros.  Bits behind the draft and the words behind a row's are not looked at."""
    n = 45
    c = Case(SHAPES["qwen36_moe"], base, n, seed=base + 1)
    seen = c.rng.random((n, n)) < 0.3
    seen[4], seen[9], seen[44] = True, False, False
    words = np.concatenate([tree_mask(seen), np.full((n, 3), 0xFFFFFFFF, np.uint32)], 1)
    words[:, 1] |= 0xFFFFFFFF << (n - 32) & 0xFFFFFFFF
    with c.context() as pa:
        c.fill(pa)
        got = pa.run_attn_tree(0, c.q, words, base, gate=c.gate)
        c.check(got, seen=seen, what="pattern")
        if base == 0:
            assert not got[9].any() and not got[44].any()


def test_one_row_gives_its_bits_back():
    """A column that sees one row alone: the value row, exactly."""
    c = Case(SHAPES["qwen3_1p7b"], 0, 40, seed=3)
    with c.context() as pa:
        c.fill(pa)
        got = pa.run_attn_tree(0, c.q, np.eye(40, dtype=bool), 0)
    assert np.array_equal(got, np.repeat(c.v, c.cfg["n_heads"] // c.cfg["n_kv_heads"], axis=1))


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("base,n", [(50, 40), (3000, 24), (0, 9)])
def test_what_is_not_finite_reaches_those_who_see_it(base, n, value):
    """A drafted row whose k and v hold what is not finite: columns that do not see it have the bits that they have with a finite row there."""
    c = Case(SHAPES["qwen36_moe"], base, n, seed=base + n)
    bad = n // 3
    hit = c.seen[:, bad]
    assert hit.any() and not hit.all()
    with c.context() as pa:
        c.fill(pa)
        clean = pa.run_attn_tree(0, c.q, c.seen, base, gate=c.gate)
        row = O.f16_bits(np.full((1, c.cfg["n_kv_heads"], c.cfg["head_dim"]), 1.0, np.float32))
        row[0, :, 5::7] = O.f16_bits(np.float32(value))
        pa.kv_write(0, 1, base + bad, row)
        v_alone = pa.run_attn_tree(0, c.q, c.seen, base, gate=c.gate)
        pa.kv_write(0, 0, base + bad, np.full_like(row, NAN16))
        both = pa.run_attn_tree(0, c.q, c.seen, base, gate=c.gate)
    assert np.array_equal(clean[~hit], v_alone[~hit]) and np.array_equal(clean[~hit], both[~hit])
    touched = np.zeros(c.cfg["head_dim"], bool)
    touched[5::7] = True
    assert not np.isfinite(v_alone[hit][..., touched]).any() and np.isfinite(v_alone[hit][..., ~touched]).all()
    if np.isinf(value):
        assert (v_alone[hit][..., touched] == value).all()
    assert np.isnan(both[hit]).all()


def test_a_chain_is_a_verify_block():
    for shape, base, n in (("qwen36_moe", 900, 7), ("qwen3_1p7b", 5000, 16), ("qwen38_27b", 40, 3)):
        c = Case(SHAPES[shape], base, n, seed=n)
        with c.context() as pa:
            c.fill(pa)
            tree = pa.run_attn_tree(0, c.q, np.tril(np.ones((n, n), bool)), base, gate=c.gate)
            block = pa.run_attn("decode", 0, c.q, base, gate=c.gate)
        c.check(tree, seen=np.tril(np.ones((n, n), bool)), what="chain")
        assert np.abs(tree - block).max() < 1e-3                    # the bound that the verify blocks' own tests put between two orders of summation


def test_peaked_scores():
    """Scores that jump by hundreds between rows: the reference of a row is raised again and again, and far ones underflow."""
    cfg = SHAPES["qwen36_moe"]
    c = Case(cfg, 700, 19, seed=8, peak=3.0)
    k = O.f16_round(c.k * (1 + 9 * (np.arange(c.k.shape[0]) % 97 == 96))[:, None, None])
    c.k, c.parts[0] = k, O.f16_bits(k)
    with c.context() as pa:
        c.fill(pa)
        for splits in (0, 1):
            pa.set_decode_splits(splits)
            got = pa.run_attn_tree(0, c.q, c.seen, c.base, gate=c.gate)
            # scores of up to 10 times the usual size: the bound of a weight is no longer small against 1, so the rows whose bound says something are the ones compared
            ref, absolute, reach = T.tree_attention(c.q, c.k, c.v, c.base, c.seen, c.gate)
            bound = T.tree_bound(ref, absolute, reach, np.abs(c.v).max(), 719)
            assert np.isfinite(got).all() and (np.abs(got - ref) <= bound).all()


def test_strides_the_q_buffer_and_untouched_memory():
    """Columns with gaps in every operand, q from the context's buffer; what lies between and behind the output's columns stays."""
    cfg = SHAPES["qwen36_moe"]
    n, base = 6, 100
    c = Case(cfg, base, n, seed=2)
    qd = cfg["n_heads"] * cfg["head_dim"]
    gap = lambda a, by: np.concatenate([a.reshape(n, -1), np.full((n, by), np.nan, np.float32)], 1)  # noqa: E731
    with c.context() as pa:
        c.fill(pa)
        dq, dg, dm = pa.to_device(gap(c.q, 8)), pa.to_device(gap(c.gate, 4)), pa.to_device(np.concatenate([tree_mask(c.seen), np.full((n, 2), 0xFFFFFFFF, np.uint32)], 1))
        dout = pa.to_device(np.full((n + 1, qd + 12), 7.0, np.float32))
        pa.attn_tree(0, dq, qd + 8, dg, qd + 4, dm, 3, base, n, dout, qd + 12)
        pa.sync()
        out = dout.download(np.float32, (n + 1) * (qd + 12)).reshape(n + 1, qd + 12)
        c.check(out[:n, :qd].reshape(c.q.shape), what="strides")
        assert (out[:n, qd:] == 7).all() and (out[n] == 7).all()
        pa._chk(pa.L.pa_upload(pa.ctx, pa.q_buffer_ptr(), np.ascontiguousarray(c.q).ctypes.data, c.q.nbytes))
        pa.attn_tree(0, None, 0, dg, qd + 4, dm, 3, base, n, dout, qd + 12)
        pa.sync()
        assert np.array_equal(dout.download(np.float32, (n + 1) * (qd + 12)).reshape(n + 1, qd + 12), out)


def test_the_last_rows_of_a_cache_and_the_same_bits_twice():
    cfg = SHAPES["qwen3_1p7b"]
    c = Case(cfg, 1990, 10, seed=1, more=0)
    with c.context() as pa:
        pa.layer_alloc(0)
        pa.kv_write(0, 0, 0, c.parts[0]); pa.kv_write(0, 1, 0, c.parts[1])
        a, b = (pa.run_attn_tree(0, c.q, c.seen, c.base) for _ in range(2))
        c.check(a, what="last rows")
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_refusals():
    cfg = SHAPES["qwen36_moe"]
    qd = cfg["n_heads"] * cfg["head_dim"]
    with PooledAttn(cfg, 200, n_layers=2, max_cols=40) as pa:
        pa.layer_alloc(0)
        d = pa.alloc(40 * qd * 8)
        m, out = pa.alloc(4096), pa.alloc(40 * qd * 8)
        good = dict(layer=0, q=d.ptr, qs=qd, g=None, gs=0, m=m.ptr, ms=2, base=100, n=40, out=out.ptr, os=qd, dt=PA_OUT_F32)

        def call(**change):
            a = dict(good, **change)
            return pa.L.pa_attn_tree(pa.ctx, a["layer"], a["q"], a["qs"], a["g"], a["gs"], a["m"], a["ms"], a["base"], a["n"], a["out"], a["os"], a["dt"])
        for change in (dict(layer=1), dict(layer=2), dict(n=0), dict(n=41), dict(base=161), dict(base=0xFFFFFFFF), dict(m=None), dict(out=None), dict(ms=1), dict(ms=0), dict(qs=qd - 4), dict(qs=qd + 2),
                       dict(os=qd - 4), dict(os=qd + 1), dict(g=d.ptr, gs=qd - 4), dict(g=d.ptr, gs=qd + 3), dict(g=d.ptr + 8, gs=qd), dict(q=d.ptr + 4), dict(out=out.ptr + 8), dict(m=m.ptr + 2),
                       dict(dt=2), dict(out=d.ptr), dict(out=d.ptr + 16), dict(q=None, out=pa.q_buffer_ptr()), dict(g=out.ptr + 4096, gs=qd), dict(m=out.ptr + 64)):
            assert call(**change) == PA_ERR_INVALID, change
            assert b"pa_attn_tree: " in pa.L.pa_last_error(pa.ctx), change
        assert call() == 0
        pa.sync()
        assert pa.L.pa_attn_tree(None, 0, None, 0, None, 0, None, 0, 0, 1, None, 0, 0) == PA_ERR_INVALID
