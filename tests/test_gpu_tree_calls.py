"""Calls around a draft tree that are refused, on the GPU: contexts whose columns have to have the bits of one-column decodes, norm weights in
buffers that the pre-step writes."""
import numpy as np
import pytest
from oracle import attn_oracle as O
from pooled_amd.capi import PooledAttn, PaError, PA_ERR_INVALID, PA_ERR_UNSUPPORTED
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


def test_norm_weights_in_the_buffers_that_the_pre_step_writes():
    n = 4
    for norm in (True, False):                            # without the norm the weights are not looked at
        cfg = dict(SHAPES["qwen36_moe"], qk_norm=norm)
        d = O.make_inputs(cfg, 0, n, 1)
        with PooledAttn(cfg, 64, n_layers=1, max_cols=n) as pa:
            pa.layer_alloc(0)
            q, k, v, qw, kw = (pa.to_device(d[x]) for x in ("qraw", "kraw", "vraw", "qw", "kw"))
            pos = pa.to_device(np.arange(n, dtype=np.uint32))
            for buf in (pa.q_buffer_ptr(), pa.gate_buffer_ptr()):
                for at in (0, 1):
                    for off in (64, n * pa.q_dim * 4 - 4):
                        w = [qw.ptr, kw.ptr]
                        w[at] = buf + off
                        rc = pa.L.pa_glue_kv_at(pa.ctx, 0, q.ptr, d["qraw"].shape[1], k.ptr, d["kraw"].shape[1], v.ptr, d["vraw"].shape[1], w[0], w[1], pos.ptr, n, 0, n)
                        assert rc == (PA_ERR_INVALID if norm else 0)
                        if norm:
                            assert b"pa_glue_kv_at: " in pa.L.pa_last_error(pa.ctx)
            pa.sync()
