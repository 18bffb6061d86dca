"""Arguments of the delta rule's entry points that a call does not use, and outputs of the pre-step beside one another."""
import numpy as np
import pytest
from pooled_amd.capi import PooledAttn, PaError, PA_ERR_INVALID
from test_gpu_delta import CTX, Case, Part, bits

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


def test_outputs_of_the_pre_step_share_nothing_but_may_interleave():
    """Two outputs in the same place are refused; the three of a column side by side in one buffer have the bits of outputs in buffers of their own."""
    n, nk, nv, hk, hv = 6, 1, 4, 64, 32
    ch = 2 * nk * hk + nv * hv
    rng = np.random.default_rng(0)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    with PooledAttn(CTX, 64, max_cols=8) as pa:
        dn = pa.delta(dict(n_k_heads=nk, n_v_heads=nv, head_k=hk, head_v=hv, conv_width=4))
        x, w, a, b, al, dt = (pa.to_device(t) for t in (f(n, ch), f(ch, 4), f(n, nv), f(n, nv), f(nv), f(nv)))
        wide = ch + 2 * nv
        one, out, g, beta = (pa.to_device(np.zeros((n, m), np.float32)) for m in (wide, ch, nv, nv))

        def run(out, os, g, beta, gs):
            pa.delta_glue(dn, 0, x, ch, w, None, a, b, nv, al, dt, n, 0, out, os, g, beta, gs)
        run(out, ch, g, beta, nv)
        run(one, wide, Part(one, 4 * ch), Part(one, 4 * (ch + nv)), wide)
        pa.sync()
        got = one.download(np.float32, n * wide).reshape(n, wide)
        for part, buf in ((got[:, :ch], out), (got[:, ch:ch + nv], g), (got[:, ch + nv:], beta)):
            assert np.array_equal(bits(part), bits(buf.download(np.float32, part.size).reshape(part.shape)))
        for bad in ((out, ch, g, g, nv), (out, ch, g, Part(g, 4), nv), (out, ch, g, Part(g, 4 * nv), nv), (out, ch, out, beta, nv), (out, ch, g, Part(out, 4 * (ch - 1)), nv),
                    (one, wide, Part(one, 4 * (ch - 1)), Part(one, 4 * (ch + nv)), wide), (one, wide, Part(one, 4 * ch), Part(one, 4 * (ch + 1)), wide)):
            with pytest.raises(PaError) as e:
                run(*bad)
            assert e.value.code == PA_ERR_INVALID and "two outputs" in str(e.value)
