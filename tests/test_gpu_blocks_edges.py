"""Calls at the borders of what the delta rule and the experts take: keys whose squares are subnormal, inputs that lie in a state, passes wider than the experts' scratch."""
import numpy as np
import pytest
from oracle import blocks_oracle as B
from pooled_amd.capi import PooledAttn, PaError, PA_ERR_INVALID, PA_OUT_F16, PA_OUT_F32, PA_W_F32, PA_W_Q4_0, PA_W_Q8_0
from test_gpu_delta import CTX, Case, Part, bits, close, step_tol
from test_gpu_moe import Layer, close as moe_close

pytestmark = pytest.mark.gpu


class Bare:
    def __init__(self, ptr):
        self.ptr = ptr


@pytest.mark.parametrize("kind,n", [("decode", 5), ("prefill", 70)])
def test_tiny_keys_without_eps(kind, n):
    """eps = 0 and keys and queries of 5e-21 a component: the sum of 128 squares of 2.5e-41 is subnormal, its own rounding half of 2^-149 a square, 2.8e-5 of it at most, so a
    length is off by 1.4e-5 at most; a token has two of k and one of q on its way, carried on like the rule's own roundings."""
    c = Case(n, seed=5)
    for a in (c.q, c.k):
        a *= np.float32(5e-21) / np.sqrt((a ** 2).mean(-1, keepdims=True))
    room = 3 * 1.4e-5 * (1 + n ** 0.5)
    with PooledAttn(CTX, 64, max_cols=128) as pa:
        dn = pa.delta(dict(n_k_heads=c.nk, n_v_heads=c.nv, head_k=c.hk, head_v=c.hv, eps=0.0))
        pa.delta_write(dn, 0, 0, c.state)
        c.upload(pa)
        out, state = c.call(pa, dn, kind), c.read(pa, dn)
    ref, ref_state = B.delta_rule(c.q, c.k, c.v, c.g, c.beta, c.state, eps=0.0)
    close(out, ref, room + 8 * step_tol(n), "out", (0, 2))
    close(state, ref_state, room + 8 * step_tol(n), "state", (1, 2))


@pytest.mark.parametrize("kind,n", [("decode", 6), ("prefill", 70)])
def test_zero_query_without_eps_is_nan_for_its_token_alone(kind, n):
    """0 / sqrt(0): the token's outputs of that q head, and nothing else."""
    c = Case(n, seed=6)
    c.q[3, 1] = 0.0
    with PooledAttn(CTX, 64, max_cols=128) as pa:
        dn = pa.delta(dict(n_k_heads=c.nk, n_v_heads=c.nv, head_k=c.hk, head_v=c.hv, eps=0.0))
        pa.delta_write(dn, 0, 0, c.state)
        c.upload(pa)
        out, state = c.call(pa, dn, kind), c.read(pa, dn)
    nan = np.zeros(out.shape, bool)
    nan[3, c.nv // 2:] = True                          # k head 1 serves the second half of the v heads
    assert np.array_equal(np.isnan(out), nan) and np.all(np.isfinite(state))
    c.q[3, 1] = 1.0
    _, ref_state = B.delta_rule(c.q, c.k, c.v, c.g, c.beta, c.state, eps=0.0)
    close(state, ref_state, 8 * step_tol(n), "state", (1, 2))


def test_inputs_in_the_state_are_refused():
    with PooledAttn(CTX, 32, max_cols=4) as pa:
        dn = pa.delta(dict(n_k_heads=1, n_v_heads=2, head_k=64, head_v=32, conv_width=4, n_layers=2))
        buf, out = pa.to_device(np.zeros(4096, np.float32)), pa.alloc(4096)
        S, conv = Bare(pa.delta_state_ptr(dn, 0, 0)), Bare(pa.delta_state_ptr(dn, 0, 1))
        for bad in range(5):
            a = [buf] * 5
            a[bad] = S
            with pytest.raises(PaError) as e:
                pa.delta_decode(dn, 0, a[0], 64, a[1], 64, a[2], 64, a[3], a[4], 2, 2, 1, out, 64)
            assert e.value.code == PA_ERR_INVALID and "state" in str(e.value)
            if bad:                                    # without an output q is not looked at
                with pytest.raises(PaError):
                    pa.delta_decode(dn, 0, None, 0, a[1], 64, a[2], 64, a[3], a[4], 2, 2, 1, None, 64)
        with pytest.raises(PaError) as e:
            pa.delta_decode(dn, 0, buf, 64, buf, 64, buf, 64, buf, buf, 2, 2, 1, S, 64)
        assert e.value.code == PA_ERR_INVALID
        pa.delta_decode(dn, 1, Part(buf, 0), 64, S, 64, buf, 64, buf, buf, 2, 2, 1, out, 64)      # another layer's state is memory like any other
        with pytest.raises(PaError) as e:
            pa.delta_glue(dn, 0, conv, 192, buf, None, buf, buf, 2, buf, buf, 2, 2, out, 192, Part(out, 2048), Part(out, 2560), 2)
        assert e.value.code == PA_ERR_INVALID and "state" in str(e.value)


@pytest.mark.parametrize("kind", [PA_W_F32, PA_W_Q8_0, PA_W_Q4_0])
def test_experts_over_more_tokens_than_the_scratch_holds(kind):
    """1100 tokens, in place: against the oracle, and the last of them with the bits of a call of their own."""
    n = 1100
    L = Layer(dim=64, ffn=32, E=9, top_k=2, kind=kind, seed=31)
    x = (L.rng.standard_normal((n, L.dim)) * 2).astype(np.float32)
    with PooledAttn(CTX, 64, max_cols=1200) as pa:
        h = L.handle(pa)
        y, ids, w = L.call(pa, h, x)
        ref, rids, _ = L.oracle(x)
        moe_close(y, x, ref)
        assert np.array_equal(ids, rids)
        y2, ids2, w2 = L.call(pa, h, x[-7:])
        assert np.array_equal(bits(y[-7:]), bits(y2)) and np.array_equal(ids[-7:], ids2) and np.array_equal(bits(w[-7:]), bits(w2))
        y3, _, _ = L.call(pa, h, x, in_place=True)
        assert np.array_equal(bits(y3), bits(y))


# heads and value columns that take 16 columns a workgroup, and as many as take 32
@pytest.mark.parametrize("nv,hv", [(4, 96), (36, 128)])
@pytest.mark.parametrize("hk", [64, 128])
@pytest.mark.parametrize("n,out", [(64, "f32"), (65, "f16"), (191, "f32"), (130, None)])
def test_prefill_of_few_and_many_heads(nv, hv, hk, n, out):
    c = Case(n, nk=nv // 2, nv=nv, hk=hk, hv=hv, seed=n + hk, fused=n == 191)
    with PooledAttn(CTX, 64, max_cols=256) as pa:
        dn = c.handle(pa)
        pa.delta_write(dn, 0, 0, c.state)
        c.upload(pa)
        got, state = c.call(pa, dn, "prefill", out=out is not None, dtype=PA_OUT_F16 if out == "f16" else PA_OUT_F32), c.read(pa, dn)
    ref, ref_state = c.oracle()
    tol = 8 * step_tol(n)
    close(state, ref_state, tol, "state", (1, 2))
    if out:
        close(got, ref, tol + (2.0 ** -11 if out == "f16" else 0), "out", (0, 2))


@pytest.mark.parametrize("nv,hv", [(4, 96), (36, 128)])
@pytest.mark.parametrize("hk", [64, 128])
@pytest.mark.parametrize("where", [(0,), (1, 2), (3,), (0, 1, 2, 3), (0, 2)])
def test_chunks_that_go_token_by_token_among_others(nv, hv, hk, where):
    """Chunks with a key of length 1.5 in some heads (no normalisation), in front of, between and behind ordinary ones, the last of 7 columns.  A state may grow by such a token:
    the factor is |1 - beta |k|^2| <= 1.25 at most, so its error too, and there is one such token a chunk."""
    n = 3 * 64 + 7
    c = Case(n, nk=nv // 2, nv=nv, hk=hk, hv=hv, seed=100 + sum(where), l2norm=False)
    for chunk in where:
        c.k[64 * chunk + 5 - 3 * (chunk == 3), ::2] *= 1.5
    with PooledAttn(CTX, 64, max_cols=256) as pa:
        dn = c.handle(pa)
        pa.delta_write(dn, 0, 0, c.state)
        c.upload(pa)
        got, state = c.call(pa, dn, "prefill"), c.read(pa, dn)
    ref, ref_state = c.oracle()
    tol = 8 * step_tol(n) * 1.25 ** len(where)
    close(got, ref, tol, "out", (0, 2))
    close(state, ref_state, tol, "state", (1, 2))


class Wide:
    """n columns with `stride` floats from one to the next, on the device; only the columns themselves are touched."""

    def __init__(self, pa, a, stride):
        self.pa, self.n, self.w, self.stride = pa, a.shape[0], a.shape[1], stride
        self.buf = pa.alloc((self.n - 1) * stride * 4 + self.w * 4)
        self.ptr = self.buf.ptr
        for i in range(self.n):
            row = np.ascontiguousarray(a[i], np.float32)
            pa._chk(pa.L.pa_upload(pa.ctx, self.ptr + 4 * i * stride, row.ctypes.data, row.nbytes))

    def read(self):
        a = np.empty((self.n, self.w), np.float32)
        for i in range(self.n):
            self.pa._chk(self.pa.L.pa_download(self.pa.ctx, a[i].ctypes.data, self.ptr + 4 * i * self.stride, a[i].nbytes))
        return a


@pytest.mark.parametrize("call,n,stride", [("decode", 17, 1 << 26), ("prefill", 260, 1 << 22), ("prefill", 70, (1 << 24) + 4)])
def test_delta_columns_past_32_bits(call, n, stride):
    """The last columns of v and of the output lie 2^32 bytes or more behind the first; strides of more than 2^22 floats go token by token.  The bits are those of dense columns."""
    assert (n - 1) * stride * 4 >= 1 << 32
    c = Case(n, nk=1, nv=2, hk=64, hv=32, seed=n, pad=0)
    col = c.nv * c.hv
    with PooledAttn(CTX, 64, max_cols=512) as pa:
        dn = pa.delta(dict(n_k_heads=1, n_v_heads=2, head_k=64, head_v=32, n_layers=2))
        flat = lambda a: np.ascontiguousarray(a.reshape(n, -1))  # noqa: E731
        q, k, v, g, b = (pa.to_device(flat(a)) for a in (c.q, c.k, c.v, c.g, c.beta))
        dense = pa.to_device(np.zeros((n, col), np.float32))
        wv, wo = Wide(pa, flat(c.v), stride), Wide(pa, np.zeros((n, col), np.float32), stride)
        for layer, (dv, vs, do, os) in enumerate(((v, col, dense, col), (wv, stride, wo, stride))):
            pa.delta_write(dn, layer, 0, c.state)
            if call == "decode":
                pa.delta_decode(dn, layer, q, 64, k, 64, dv, vs, g, b, 2, n, n, do, os)
            else:
                pa.delta_prefill(dn, layer, q, 64, k, 64, dv, vs, g, b, 2, n, do, os)
        pa.sync()
        got, ref = wo.read(), dense.download(np.float32, n * col).reshape(n, col)
        s0, s1 = pa.delta_read(dn, 0, 0), pa.delta_read(dn, 1, 0)
    if call == "prefill" and stride > 1 << 22:
        close(got, ref, 9 * step_tol(n), "out", (0,))
        close(s1, s0, 9 * step_tol(n), "state", (0,))
    else:
        assert np.array_equal(bits(got), bits(ref)) and np.array_equal(bits(s0), bits(s1))


def test_experts_columns_past_32_bits():
    n, stride = 33, 1 << 26
    L = Layer(dim=96, ffn=32, E=7, top_k=2, kind=PA_W_Q4_0, seed=3)
    x = (L.rng.standard_normal((n, L.dim)) * 2).astype(np.float32)
    with PooledAttn(CTX, 64, max_cols=64) as pa:
        h = L.handle(pa)
        ref, _, _ = L.call(pa, h, x)
        wx = Wide(pa, x, stride)
        pa.moe_layer(h, pa.to_device(L.norm), wx, stride, n, wx, stride)
        pa.sync()
        assert np.array_equal(bits(wx.read()), bits(ref))
