"""What is not finite in rows of the context (pa_attn_tree) on the GPU: every column sees those rows, so it reaches every column, in whatever tile it lies and in front of whatever draft."""
import numpy as np
import pytest
from oracle import attn_oracle as O
from oracle import tree_oracle as T
from test_gpu_tree import Case
from helpers import SHAPES

pytestmark = pytest.mark.gpu
NUMBERS = [np.inf, -np.inf, np.nan]


def rows_of(base):
    """The context's last row, the first of the tile that the draft begins in, one between, and the last of the tile in front."""
    first = base // 32 * 32
    return sorted({base - 1, first, (first + base) // 2} | ({first - 1} if first else set()))


def run(c, pa, splits):
    pa.set_decode_splits(splits)
    return pa.run_attn_tree(0, c.q, c.seen, c.base, gate=c.gate)


def oracle(c):
    ref, absolute, reach = T.tree_attention(c.q, c.k, c.v, c.base, c.seen, c.gate)
    return ref, T.tree_bound(ref, absolute, reach, np.abs(c.v).max(), c.base + c.n, bool(c.cfg.get("kv_q8")))


def check(got, ref, bound, touched, value):
    """touched [hd]: the dims that hold `value` in a row; the others are what they are without."""
    hit = got[..., touched]
    assert (np.isnan(hit) if np.isnan(value) else hit == value).all()
    assert (np.abs(got - ref) <= bound)[..., ~touched].all()


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("shape", ["qwen36_moe", "qwen3_1p7b"])
@pytest.mark.parametrize("base,n", [(50, 40), (3000, 24), (33, 5), (95, 70)])
def test_f16_rows(shape, base, n, splits):
    c = Case(SHAPES[shape], base, n, seed=base + n)
    want, touched = oracle(c), np.zeros(c.cfg["head_dim"], bool)
    touched[5::7] = True
    with c.context() as pa:
        c.fill(pa)
        for at in rows_of(base):
            for value in NUMBERS:
                print("context row", shape, base, n, splits, at, value, flush=True)
                row = c.parts[1][at:at + 1].copy()
                row[..., touched] = O.f16_bits(np.float32(value))
                pa.kv_write(0, 1, at, row)
                check(run(c, pa, splits), *want, touched, value)
            pa.kv_write(0, 1, at, c.parts[1][at:at + 1])


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("shape", ["qwen36_moe", "qwen3_1p7b"])
@pytest.mark.parametrize("base,n", [(50, 40), (3000, 24)])
def test_int8_rows(shape, base, n, splits):
    """The same through a block's scale; a scale that takes values out of f16's range (127 x 600) makes them infinite wherever the row lies."""
    c = Case(dict(SHAPES[shape], kv_q8=True), base, n, seed=base + n)
    want, touched = oracle(c), np.zeros(c.cfg["head_dim"], bool)
    touched[32:64] = True
    with c.context() as pa:
        c.fill(pa)
        for at in rows_of(base):
            for value, scale, number in ((np.nan, np.nan, 5), (np.inf, 600.0, 127), (-np.inf, 600.0, -127)):
                print("context row, int8", shape, base, n, splits, at, value, scale, flush=True)
                row, sc = c.parts[1][at:at + 1].copy(), c.parts[3][at:at + 1].copy()
                row[..., touched], sc[..., 1] = number, scale
                pa.kv_write(0, 1, at, row); pa.kv_write(0, 3, at, sc)
                check(run(c, pa, splits), *want, touched, value)
            pa.kv_write(0, 1, at, c.parts[1][at:at + 1]); pa.kv_write(0, 3, at, c.parts[3][at:at + 1])


def test_a_row_of_the_context_and_a_drafted_one():
    """Both in one tile: the context's reaches every column, the drafted one those that see it."""
    c = Case(SHAPES["qwen36_moe"], 50, 40, seed=4)
    bad = 9                                              # in the tile of rows 32 .. 63, as row 40 of the context is
    sees = c.seen[:, bad]
    assert sees.any() and not sees.all()
    with c.context() as pa:
        c.fill(pa)
        for at, dim in ((40, 3), (50 + bad, 8)):
            row = c.parts[1][at:at + 1].copy()
            row[..., dim] = O.f16_bits(np.float32(np.inf))
            pa.kv_write(0, 1, at, row)
        for splits in (1, 3):
            got = run(c, pa, splits)
            finite = np.isfinite(got)
            assert not finite[..., 3].any() and not finite[sees][..., 8].any() and finite[~sees][..., 8].all()
            assert np.delete(finite, [3, 8], axis=2).all()
