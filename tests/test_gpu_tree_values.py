"""Numbers that pa_attn_tree holds in f16, on the GPU against the oracle in 64 bits: int8 rows' values from the smallest to the largest scales, and queries."""
import numpy as np
import pytest
from oracle import attn_oracle as O
from oracle import tree_oracle as T
from test_gpu_tree import Case
from test_tree_rules import tree_rule
from helpers import SHAPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("base,n,splits", [(40, 9, 1), (40, 9, 2), (500, 33, 0)])
def test_int8_rows_of_any_size(shape, base, n, splits):
    """A block of 32 dims of V is up to 4e4 to 3e-6 large, one size a block; keys as they are.  A value is its scale times a whole number, rounded once to f16: off by 2^-11 of itself and 2^-21 more
    for the parts of the scale, or, where f16 is subnormal, by 2^-25 for either of product and sum, 2^-24 in all; an output, a mean of values, by no more."""
    c = Case(dict(SHAPES[shape], kv_q8=True), base, n, seed=base + n, peak=0.1)
    hd = c.cfg["head_dim"]
    size = np.repeat(10.0 ** np.linspace(4.6, -5.5, hd // 32), 32)
    val, sc = O.q8_quantize((c.v * (size / 4)).astype(np.float32))
    c.parts[1], c.parts[3], c.v = val, sc, O.q8_dequantize(val, sc)
    assert np.abs(c.v).max() < 65000
    with c.context() as pa:
        c.fill(pa)
        pa.set_decode_splits(splits)
        got = pa.run_attn_tree(0, c.q, c.seen, base, gate=c.gate)
    ref, absolute, reach = T.tree_attention(c.q, c.k, c.v, base, c.seen, c.gate)
    heads = c.cfg["n_heads"] // c.cfg["n_kv_heads"]
    bound = T.tree_bound(ref, absolute, reach, np.repeat(np.abs(c.v).max(0), heads, axis=0), base + n, True) + 2.0 ** -24
    off = np.abs(got - ref)
    for b in range(hd // 32):
        at = np.s_[..., 32 * b:32 * b + 32]
        print("int8 %s base %d, values up to %.1e: off by %.1e of outputs of %.1e, %.1f %% of the bound" % (
            shape, base, np.abs(c.v[at]).max(), off[at].max(), np.abs(ref[at]).max(), 100 * (off[at] / bound[at]).max()), flush=True)
    assert (off <= bound).all()


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("scale", [2e-7, 3e-6, 1.1e-5, 3e-5, 7e-4, 0.02, 3.0, 300.0])
def test_one_int8_row_comes_back(shape, scale):
    """A column that sees one row alone gives that row's values: whole number times scale, rounded to f16."""
    cfg = dict(SHAPES[shape], kv_q8=True)
    c = Case(cfg, 0, 20, seed=5)
    c.gate = None
    c.parts[3] = (c.parts[3] * 0 + scale * np.linspace(1.0, 1.5, c.parts[3].shape[-1])).astype(np.float32)
    with c.context() as pa:
        c.fill(pa)
        got = pa.run_attn_tree(0, c.q, np.eye(20, dtype=bool), 0)
    want = np.repeat(O.q8_dequantize(c.parts[1], c.parts[3]).astype(np.float64), cfg["n_heads"] // cfg["n_kv_heads"], axis=1)
    off = np.abs(got - want)
    print("scale %.1e: off by up to %.2e of a value" % (scale, (off / np.maximum(np.abs(want), scale)).max()), flush=True)
    assert (off <= np.abs(want) * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -24).all()


@pytest.mark.parametrize("value", [np.inf, -np.inf])
@pytest.mark.parametrize("base,n,at,splits", [(50, 40, 49, 1), (50, 40, 5, 2), (3000, 24, 2999, 3), (50, 40, 60, 1), (50, 40, 60, 3)])
def test_an_infinite_int8_scale(base, n, at, splits, value):
    """Whole numbers times infinity: infinities of their sign (rows of the context and drafted ones alike), for the columns that see the row."""
    c = Case(dict(SHAPES["qwen36_moe"], kv_q8=True), base, n, seed=3)
    row, sc = c.parts[1][at:at + 1].copy(), c.parts[3][at:at + 1].copy()
    row[..., 64:96], sc[..., 2] = 5 if value > 0 else -5, np.inf
    c.parts[1][at], c.parts[3][at] = row[0], sc[0]
    sees = c.seen[:, at - base] if at >= base else np.ones(n, bool)
    with c.context() as pa:
        c.fill(pa)
        pa.set_decode_splits(splits)
        got = pa.run_attn_tree(0, c.q, c.seen, base, gate=c.gate)
    assert (got[sees][..., 64:96] == value).all() and np.isfinite(got[~sees]).all() and np.isfinite(np.delete(got, np.arange(64, 96), axis=2)).all()


def long_queries(c):
    """Long queries at right angles to the keys that their column sees, but for a small part: rounded to f16, their scores would be off by some hundredths."""
    G, hd = c.cfg["n_heads"] // c.cfg["n_kv_heads"], c.cfg["head_dim"]
    for g in range(c.cfg["n_kv_heads"]):
        for col in range(c.n):
            K = c.k[np.concatenate([np.ones(c.base, bool), c.seen[col]]), g].astype(np.float64)
            assert 0 < K.shape[0] < hd
            back, far = np.linalg.pinv(K), 20 * c.rng.standard_normal((hd, G))
            c.q[col, g * G:g * G + G] = (far - back @ (K @ far) + back @ (np.sqrt(hd) * c.rng.standard_normal((K.shape[0], G)))).T


def check_queries(c, splits, what):
    """q counts to 2^-22 of itself (its f16 and what that leaves).  What is left are P and f32 sums, and an output of f16 or a part of the like: at most four roundings of half a step, 2^-11, that
    add in squares (as in test_gpu_tree_run.check_some): 2^-10 of the norm."""
    with c.context() as pa:
        c.fill(pa)
        pa.set_decode_splits(splits)
        got = pa.run_attn_tree(0, c.q, c.seen, c.base, gate=c.gate)
    ref = T.tree_attention(c.q, c.k, c.v, c.base, c.seen, c.gate)[0]
    norm = np.sqrt(((got - ref) ** 2).sum() / (ref ** 2).sum())
    print("%s base %d n %d: %.2e of the norm" % (what, c.base, c.n, norm), flush=True)
    assert norm <= 2.0 ** -10


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("base,splits", [(0, 0), (3, 0), (40, 1), (59, 2)])
def test_queries_of_small_drafts(shape, base, splits):
    """Up to eight stacked rows, as in a verify block of the same columns."""
    cfg = SHAPES[shape]
    for n in sorted({1, 8 // (cfg["n_heads"] // cfg["n_kv_heads"])}):
        c = Case(cfg, base, n, seed=base + n)
        long_queries(c)
        check_queries(c, splits, "small draft " + shape)


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("base,n,splits", [(0, 5, 0), (20, 9, 1), (20, 9, 2), (7, 24, 0), (40, 40, 3), (64, 60, 4)])
def test_queries_of_more_rows(shape, base, n, splits):
    """One block of rows a wave, and two of heads of 128."""
    cfg = SHAPES[shape]
    if cfg["head_dim"] == 256:
        assert tree_rule(cfg, base, n, splits)[0] == 1
    c = Case(cfg, base, n, seed=base + n)
    long_queries(c)
    check_queries(c, splits, "draft " + shape)


@pytest.mark.parametrize("splits", [0, 3])
def test_queries_of_two_blocks_a_wave(splits):
    """Heads of 128 in a draft so wide that its plan has them, each column seeing a few rows."""
    cfg, n = dict(n_heads=64, n_kv_heads=1, head_dim=128, n_rot=64, rope_theta=1e6, eps=1e-6, qk_norm=True, gate=False), 1000
    assert tree_rule(cfg, 0, n, splits)[0] == 2
    c = Case(cfg, 0, n, seed=n)
    c.seen = c.rng.random((n, n)) < 0.006
    c.seen[np.arange(n), np.arange(n)] = True
    long_queries(c)
    check_queries(c, splits, "two blocks a wave,")


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("base,n,splits", [(20, 9, 1), (40, 9, 2), (90, 17, 3), (300, 40, 7)])
def test_parts_of_a_mean_are_kept_in_f32(shape, base, n, splits, q8):
    """Queries of zeros weigh every seen row alike, exactly, over values in [1, 2) that f16 holds: an output is a mean, whose sums, and those of the splits' parts, are off by 2^-24 of themselves for every
    row and every part at most, and by a few of that for reciprocal, product and gate (2^-22 for the hardware's reciprocal and exponential)."""
    c = Case(dict(SHAPES[shape], kv_q8=q8), base, n, seed=base)
    c.q[:] = 0
    if q8:
        c.parts[1] = (c.parts[1] & 63 | 64).astype(np.int8)
        c.parts[3][:] = 2.0 ** -6
        c.v = O.q8_dequantize(c.parts[1], c.parts[3])
    else:
        c.v = O.f16_round((1 + np.abs(c.v) % 1).astype(np.float32))
        c.parts[1] = O.f16_bits(c.v)
    assert c.v.min() >= 1 and c.v.max() <= 2
    with c.context() as pa:
        c.fill(pa)
        pa.set_decode_splits(splits)
        got = pa.run_attn_tree(0, c.q, c.seen, base, gate=c.gate)
    ref = T.tree_attention(c.q, c.k, c.v, base, c.seen, c.gate)[0]
    off = np.abs(got / ref - 1).max()
    print("mean %s%s base %d n %d in %d: off by %.2e" % (shape, " q8" if q8 else "", base, n, splits, off), flush=True)
    assert off <= (base + n + splits + 4) * 2.0 ** -24 + 2.0 ** -21
