"""The merge of a split context (pa_attn_tree) on the GPU: an infinite value in a row that every column sees comes out infinite, in whichever split it lies and whatever their number."""
import numpy as np
import pytest
from oracle import attn_oracle as O
from oracle import tree_oracle as T
from test_gpu_tree import Case
from helpers import SHAPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("shape", ["qwen36_moe", "qwen3_1p7b"])
@pytest.mark.parametrize("splits", [2, 3, 8, 9, 17, 31])
def test_an_infinite_value_in_any_split(shape, splits, value):
    c = Case(SHAPES[shape], 1000, 20, seed=splits)                       # 32 tiles, the draft from the last but one on
    with c.context() as pa:
        c.fill(pa)
        pa.set_decode_splits(splits)
        for at in (3, 500, 980):
            row, v = c.parts[1][at:at + 1].copy(), c.v.copy()
            row[..., 7], v[at][..., 7] = O.f16_bits(np.float32(value)), 0
            pa.kv_write(0, 1, at, row)
            got = pa.run_attn_tree(0, c.q, c.seen, c.base, gate=c.gate)
            pa.kv_write(0, 1, at, c.parts[1][at:at + 1])
            print("merge", shape, splits, at, value, flush=True)
            ref, absolute, reach = T.tree_attention(c.q, c.k, v, c.base, c.seen, c.gate)
            assert (np.isnan(got[..., 7]) if np.isnan(value) else got[..., 7] == value).all()
            assert (np.abs(got - ref) <= T.tree_bound(ref, absolute, reach, np.abs(v).max(), 1020))[..., np.arange(c.cfg["head_dim"]) != 7].all()
