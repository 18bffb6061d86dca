"""Arguments of the delta rule's entry points that a call does not use, and outputs of the pre-step beside one another."""
import numpy as np
import pytest
from pooled_amd.capi import PooledAttn
from test_gpu_delta import CTX, Case, bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_stride", [0, 1, (1 << 22) + 4, 0xFFFFFFFF])
def test_a_prefill_without_outputs_does_not_look_at_their_stride(out_stride):
    """The state has the bits of the same call with outputs, whatever the stride of the outputs that are not there."""
    c = Case(130, nk=1, nv=2, hv=32, seed=4)
    with PooledAttn(CTX, 256, max_cols=256) as pa:
        dn = c.handle(pa, n_layers=2)
        c.upload(pa)
        for layer in (0, 1):
            pa.delta_write(dn, layer, 0, c.state)
        c.call(pa, dn, "prefill")
        pa.delta_prefill(dn, 1, None, 0, c.dk, c.ks, c.dv, c.vs, c.dg, c.dbeta, c.gs, c.n, None, out_stride)
        pa.sync()
        assert np.array_equal(bits(pa.delta_read(dn, 0, 0)), bits(pa.delta_read(dn, 1, 0)))
