"""Calls around a draft tree that are refused, on the GPU: contexts whose columns have to have the bits of one-column decodes."""
import numpy as np
import pytest
from pooled_amd.capi import PaError, PA_ERR_UNSUPPORTED
from test_gpu_tree import Case
from helpers import SHAPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [False, True])
def test_a_context_of_exact_columns(q8):
    """PA_FLAG_VERIFY_EXACT promises the bits of one-column decodes, which a tree's stacked columns do not have; verify blocks of the same context go on."""
    c = Case(dict(SHAPES["qwen36_moe"], kv_q8=q8, verify_exact=True), 100, 5, seed=1)
    with c.context() as pa:
        c.fill(pa)
        for seen in (c.seen, np.tril(np.ones((5, 5), bool))):
            with pytest.raises(PaError) as e:
                pa.run_attn_tree(0, c.q, seen, 100, gate=c.gate)
            assert e.value.code == PA_ERR_UNSUPPORTED and "pa_attn_tree: " in str(e.value) and "VERIFY_EXACT" in str(e.value)
        assert np.isfinite(pa.run_attn("decode", 0, c.q, 100, gate=c.gate)).all()
