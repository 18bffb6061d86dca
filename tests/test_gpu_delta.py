"""The gated delta rule and its pre-step through the C ABI against the 64-bit oracle.

Tolerances, relative to the 2-norm of a head's result.  A rounding to f32 is off by at most 2^-24.  One token of the rule is two dot products of
head_k <= 128 values (per lane at most 16 products one after another, then 4 levels), norms of q and k (the same, halved by the square root), two scalings and an update: at
most 24 roundings lie on any path from an input to an output of the token.  The error of a state is carried on, never amplified (0 <= beta <= 1 over unit keys and decays <= 1 are
contractions), and the roundings of different tokens are independent, so after n tokens it is at most 24 x 2^-24 x (1 + sqrt(n)) of the norms that meet: STEP(n).  The
chunked form works on f16 pairs of 22 bits (hi + lo, off by 2^-23 at most), drops the product of the two low halves (2^-22) and meets three products on the way: 8 x STEP(n).
f16 results add half a step, 2^-11, per value."""
import ctypes

import numpy as np
import pytest
from oracle import blocks_oracle as B
from pooled_amd import capi
from pooled_amd.capi import PooledAttn, PaError, PA_ERR_INVALID, PA_ERR_UNSUPPORTED, PA_OUT_F16, PA_OUT_F32

pytestmark = pytest.mark.gpu
CTX = dict(n_heads=1, n_kv_heads=1, head_dim=128, n_rot=64, rope_theta=1e6, eps=1e-6)


def step_tol(n):
    return 24 * 2.0 ** -24 * (1 + n ** 0.5)


class Part:
    """Part of a device buffer, for calls that take columns of a wider array."""

    def __init__(self, buf, offset):
        self.ptr = buf.ptr + offset


class Case:
    """Inputs of one call and the calls themselves; every column has `pad` floats behind it, filled with NaN, and the output a canary."""

    def __init__(self, n, nk=2, nv=4, hk=128, hv=128, seed=0, pad=4, fused=False, l2norm=True, scale=0.0, state=0.1):
        rng = np.random.default_rng(seed)
        self.n, self.nk, self.nv, self.hk, self.hv, self.pad, self.fused, self.l2norm, self.scale = n, nk, nv, hk, hv, pad, fused, l2norm, scale
        silu = lambda x: x / (1 + np.exp(-x))  # noqa: E731
        f = lambda *s: silu(rng.standard_normal(s)).astype(np.float32)  # noqa: E731
        self.q, self.k, self.v = f(n, nk, hk), f(n, nk, hk), f(n, nv, hv)
        if not l2norm:
            self.q /= np.sqrt((self.q ** 2).sum(-1, keepdims=True)); self.k /= np.sqrt((self.k ** 2).sum(-1, keepdims=True)) * 1.0001
        self.g = (-np.exp(rng.uniform(0, 2.8, nv)) * np.log1p(np.exp(rng.standard_normal((n, nv)) - 4))).astype(np.float32)
        self.beta = B.sigmoid(rng.standard_normal((n, nv))).astype(np.float32)
        self.state = (state * rng.standard_normal((nv, hv, hk))).astype(np.float32)

    def oracle(self, commit=None):
        return B.delta_rule(self.q, self.k, self.v, self.g, self.beta, self.state, scale=self.scale, l2norm=self.l2norm, commit=commit)

    def handle(self, pa, n_layers=1):
        return pa.delta(dict(n_k_heads=self.nk, n_v_heads=self.nv, head_k=self.hk, head_v=self.hv, n_layers=n_layers, l2norm=self.l2norm, scale=self.scale))

    def _padded(self, a):
        a = a.reshape(self.n, -1)
        return np.concatenate([a, np.full((self.n, self.pad), np.nan, np.float32)], 1)

    def upload(self, pa):
        n = self.n
        if self.fused:                             # q, k and v are parts of one column, as the pre-step writes them
            x = self._padded(np.concatenate([a.reshape(n, -1) for a in (self.q, self.k, self.v)], 1))
            b, s, kd = pa.to_device(x), x.shape[1], self.nk * self.hk
            self.dq, self.dk, self.dv, self.qs, self.ks, self.vs = b, Part(b, 4 * kd), Part(b, 8 * kd), s, s, s
        else:
            parts = [self._padded(a) for a in (self.q, self.k, self.v)]
            self.dq, self.dk, self.dv = (pa.to_device(p) for p in parts)
            self.qs, self.ks, self.vs = (p.shape[1] for p in parts)
        gates = [self._padded(a) for a in (self.g, self.beta)]
        self.dg, self.dbeta, self.gs = pa.to_device(gates[0]), pa.to_device(gates[1]), gates[0].shape[1]

    def call(self, pa, dn, kind, layer=0, c0=0, n=None, commit=None, out=True, dtype=PA_OUT_F32):
        """Columns c0 .. c0 + n; returns them [n, nv, hv], after checking that nothing else of the output was touched."""
        n = self.n - c0 if n is None else n
        at = lambda d, s: Part(d, 4 * s * c0)  # noqa: E731
        col, elem = self.nv * self.hv, 4 if dtype == PA_OUT_F32 else 2
        stride = col + 3
        canary = np.full((n + 1, stride), 12345.0, np.float32 if elem == 4 else np.float16)
        do = pa.to_device(canary) if out else None
        args = [dn, layer, at(self.dq, self.qs) if out else None, self.qs, at(self.dk, self.ks), self.ks, at(self.dv, self.vs), self.vs, at(self.dg, self.gs), at(self.dbeta, self.gs),
                self.gs, n] + ([n if commit is None else commit] if kind == "decode" else []) + [do, stride, dtype]
        (pa.delta_decode if kind == "decode" else pa.delta_prefill)(*args)
        pa.sync()
        if not out:
            return None
        got = do.download(canary.dtype, canary.size).reshape(canary.shape)
        do.free(); pa._bufs.remove(do)
        assert np.all(got[n] == 12345.0) and np.all(got[:n, col:] == 12345.0), "wrote outside the columns"
        return got[:n, :col].reshape(n, self.nv, self.hv)

    def read(self, pa, dn, layer=0):
        return pa.delta_read(dn, layer, 0).reshape(self.nv, self.hv, self.hk)


def close(got, ref, tol, what, axis):
    """2-norm of the difference over 2-norm of the reference, per head."""
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert np.all(np.isfinite(got)), "%s: non-finite" % what
    d = np.sqrt(((got - ref) ** 2).sum(axis)) / np.maximum(np.sqrt((ref ** 2).sum(axis)), 1e-30)
    print("%s: relative error %.2e of %.2e" % (what, d.max(), tol))
    assert d.max() <= tol, "%s: relative error %.3e, tolerance %.3e" % (what, d.max(), tol)


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32 if a.dtype == np.float32 else np.uint16)


def check(c, pa, kind, dtype=PA_OUT_F32, factor=1, **kw):
    dn = c.handle(pa)
    pa.delta_write(dn, 0, 0, c.state)
    c.upload(pa)
    out, state = c.call(pa, dn, kind, dtype=dtype, **kw), c.read(pa, dn)
    ref, ref_state = c.oracle(kw.get("commit"))
    tol = factor * step_tol(c.n)
    close(out, ref, tol + (2.0 ** -11 if dtype == PA_OUT_F16 else 0), "out", (0, 2))
    close(state, ref_state, tol, "state", (1, 2))
    return out, state


SHAPES = [dict(nk=2, nv=4, hk=128, hv=128), dict(nk=1, nv=1, hk=64, hv=16), dict(nk=2, nv=6, hk=64, hv=96), dict(nk=3, nv=3, hk=128, hv=48), dict(nk=1, nv=2, hk=128, hv=512)]


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 9, 16])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_decode(shape, n):
    with PooledAttn(CTX, 32, max_cols=16) as pa:
        check(Case(n, seed=10 * n + shape, pad=4 * (n % 2), fused=n % 3 == 0, **SHAPES[shape]), pa, "decode", dtype=PA_OUT_F16 if n == 5 else PA_OUT_F32)


@pytest.mark.parametrize("n", [1, 17, 47, 48, 49, 63, 64, 65, 127, 128, 130, 191, 333, 1000, 2047, 2048, 2049, 2200])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_prefill(shape, n):
    if n > 1000 and shape not in (0, 2):
        n -= 1500                                  # 547 .. 700: the other shapes at middle lengths
    with PooledAttn(CTX, 4096, max_cols=max(n, 16)) as pa:
        check(Case(n, seed=10 * n + shape, pad=4 * (n % 2), fused=n % 3 == 0, **SHAPES[shape]), pa, "prefill", dtype=PA_OUT_F16 if n % 5 == 0 else PA_OUT_F32, factor=8)


@pytest.mark.parametrize("kind", ["decode", "prefill"])
def test_without_normalisation_and_with_a_scale_of_its_own(kind):
    with PooledAttn(CTX, 512, max_cols=256) as pa:
        check(Case(100, seed=3, l2norm=False, scale=-0.37, nk=2, nv=4, hk=64, hv=64), pa, kind, factor=8 if kind == "prefill" else 1)


def test_a_draft_has_the_bits_of_single_tokens_and_leaves_the_state():
    c = Case(7, seed=5)
    with PooledAttn(CTX, 32, max_cols=16) as pa:
        dn = c.handle(pa, n_layers=2)
        c.upload(pa)
        for layer in (0, 1):
            pa.delta_write(dn, layer, 0, c.state)
        draft = c.call(pa, dn, "decode", commit=0)
        assert np.array_equal(bits(c.read(pa, dn)), bits(c.state)), "a draft with nothing committed changed the state"
        partly = c.call(pa, dn, "decode", commit=4)
        assert np.array_equal(bits(draft), bits(partly))
        single = [c.call(pa, dn, "decode", layer=1, c0=i, n=1) for i in range(4)]
        assert np.array_equal(bits(np.concatenate(single)), bits(draft[:4])), "draft columns differ from single tokens"
        assert np.array_equal(bits(c.read(pa, dn)), bits(c.read(pa, dn, 1))), "state after four columns"
        c.call(pa, dn, "decode", c0=4, n=3, out=False)                                  # the accepted columns again, without outputs
        rest = [c.call(pa, dn, "decode", layer=1, c0=i, n=1) for i in range(4, 7)]
        assert np.array_equal(bits(np.concatenate(rest)), bits(draft[4:]))
        assert np.array_equal(bits(c.read(pa, dn)), bits(c.read(pa, dn, 1))), "state after a call without outputs"


@pytest.mark.parametrize("kind", ["decode", "prefill"])
def test_calls_go_on_from_the_state_and_repeat_their_bits(kind):
    c = Case(300, seed=6, nk=1, nv=2)
    with PooledAttn(CTX, 512, max_cols=300) as pa:
        runs = []
        for _ in range(2):
            dn = c.handle(pa)
            c.upload(pa)
            pa.delta_write(dn, 0, 0, c.state)
            outs = [c.call(pa, dn, kind, c0=a, n=b - a) for a, b in ((0, 100), (100, 101), (101, 300))]
            runs.append((np.concatenate(outs), c.read(pa, dn)))
        ref, ref_state = c.oracle()
        close(runs[0][0], ref, 8 * step_tol(300), "out", (0, 2))
        close(runs[0][1], ref_state, 8 * step_tol(300), "state", (1, 2))
        assert np.array_equal(bits(runs[0][0]), bits(runs[1][0])) and np.array_equal(bits(runs[0][1]), bits(runs[1][1]))


@pytest.mark.parametrize("kind", ["decode", "prefill"])
def test_state_without_outputs(kind):
    c = Case(150, seed=8, hv=64)
    with PooledAttn(CTX, 512, max_cols=300) as pa:
        states = []
        for out in (True, False):
            dn = c.handle(pa)
            c.upload(pa)
            pa.delta_write(dn, 0, 0, c.state)
            c.call(pa, dn, kind, out=out)
            states.append(c.read(pa, dn))
        assert np.array_equal(bits(states[0]), bits(states[1]))


def _poke(c, what):
    """Inputs at the edges of what the formulas allow."""
    n, m = c.n, c.n // 2
    if what == "emptied":
        c.g[m, 0] = -np.inf; c.g[3] = -np.inf
    elif what == "left out":
        c.beta[m:m + 5] = 0; c.beta[:, -1] = 0
    elif what == "fast decay":
        c.g[:] = -np.abs(c.g) * 200 - 5; c.g[m:] *= 1e-4
    elif what == "no decay":
        c.g[:] = 0; c.beta[:] = 1
    elif what == "zero keys":
        c.k[m:m + 3] = 0; c.q[m] = 0
    elif what == "one key":
        c.k[:] = c.k[:1]; c.g[:] *= 0.01
    elif what == "alternating keys":
        c.k[:] = c.k[:1] * np.where(np.arange(n) % 2, -1, 1)[:, None, None]; c.beta[:] = 0.99
    elif what == "beta of two":
        c.beta[:] = 2; c.g[:] = -0.02
    elif what == "growth":
        c.g[m] = 0.5; c.g[5, 0] = 1.0
    elif what == "far beta":
        c.beta[m] = 7; c.beta[9, 1] = -0.5; c.g[:] = -0.7
    elif what == "large values":
        c.v[:] *= 1e30; c.v[m] *= 1e5
    elif what == "small values":
        c.v[:] *= 1e-30; c.state[:] = 0
    elif what == "values apart":
        c.v[:, :, ::2] *= 1e-12; c.state[:, ::2] *= 1e-12
    elif what == "a jump":
        c.v[m:] *= 1e9
    elif what == "small after large":
        c.v[m:] *= 1e-9; c.g[m] = -np.inf
    else:
        raise ValueError(what)


EDGES = ["emptied", "left out", "fast decay", "no decay", "zero keys", "one key", "alternating keys", "beta of two", "growth", "far beta", "large values", "small values", "values apart",
         "a jump", "small after large"]


@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("what", EDGES)
def test_edges(what, kind):
    c = Case(150, seed=9, nk=1, nv=2, hv=32)
    _poke(c, what)
    with PooledAttn(CTX, 512, max_cols=150) as pa:
        out, state = check(c, pa, kind, factor=8 if kind == "prefill" else 1)
        if what == "values apart":                 # each value column is a recurrence of its own, whatever its neighbours' size
            ref, ref_state = c.oracle()
            close(out[:, :, ::2], ref[:, :, ::2], 8 * step_tol(c.n), "small columns", (0, 2))
            close(state[:, ::2], ref_state[:, ::2], 8 * step_tol(c.n), "small rows of the state", (1, 2))


@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("l2norm,size", [(False, 3.0), (False, 1e-5), (True, 1e4), (True, 1e-9)])
def test_keys_of_other_lengths(kind, l2norm, size):
    """Unnormalised keys longer than one (with steps that keep the rule from growing) or tiny, and normalised ones whose squares are far from eps."""
    c = Case(130, seed=11, nk=1, nv=1, hv=32, l2norm=l2norm)
    c.k *= np.float32(size); c.q *= np.float32(size)
    if not l2norm:
        c.beta *= np.float32(min(1.0, size ** -2))
    with PooledAttn(CTX, 512, max_cols=150) as pa:
        check(c, pa, kind, factor=8)


@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("where", ["v", "k", "g", "beta", "q", "inf v"])
def test_a_nan_reaches_what_the_formulas_say(kind, where):
    c = Case(140, seed=12, nk=1, nv=2, hv=32)
    t = 70
    if where in ("v", "inf v"):
        c.v[t, 1, 3] = np.nan if where == "v" else np.inf
    elif where in ("k", "q"):
        getattr(c, where)[t, 0, 5] = np.nan
    else:
        getattr(c, where)[t, 1] = np.nan
    with np.errstate(invalid="ignore"):
        ref, ref_state = c.oracle()
    with PooledAttn(CTX, 512, max_cols=150) as pa:
        dn = c.handle(pa)
        pa.delta_write(dn, 0, 0, c.state)
        c.upload(pa)
        out, state = c.call(pa, dn, kind), c.read(pa, dn)
    assert np.array_equal(np.isfinite(out), np.isfinite(ref)), "non-finite outputs elsewhere than in the oracle"
    assert np.array_equal(np.isfinite(state), np.isfinite(ref_state)), "non-finite state elsewhere than in the oracle"
    good = np.where(np.isfinite(ref), ref, 0)
    close(np.where(np.isfinite(out), out, 0), good, 8 * step_tol(c.n), "finite outputs", (0, 2))


# ---- pre-step ---------------------------------------------------------------------------------------------------------

def _glue(pa, dn, layer, x, w, bias, a, b, a_log, dt_bias, commit, pad):
    n, ch, nv = x.shape[0], x.shape[1], a.shape[1]
    wide = lambda t: np.concatenate([t, np.full((n, pad), np.nan, np.float32)], 1)  # noqa: E731
    outs = [pa.to_device(np.full((n + 1, m + pad), 777.0, np.float32)) for m in (ch, nv, nv)]
    pa.delta_glue(dn, layer, pa.to_device(wide(x)), ch + pad, pa.to_device(w), pa.to_device(bias) if bias is not None else None, pa.to_device(wide(a)), pa.to_device(wide(b)), nv + pad,
                  pa.to_device(a_log), pa.to_device(dt_bias), n, commit, outs[0], ch + pad, outs[1], outs[2], nv + pad)
    pa.sync()
    res = []
    for o, m in zip(outs, (ch, nv, nv)):
        got = o.download(np.float32, (n + 1) * (m + pad)).reshape(n + 1, m + pad)
        assert np.all(got[n] == 777.0) and np.all(got[:n, m:] == 777.0), "wrote outside the columns"
        res.append(got[:n, :m])
    return res


@pytest.mark.parametrize("width", [1, 2, 3, 4])
@pytest.mark.parametrize("n,commit", [(1, 1), (1, 0), (2, 1), (3, 3), (7, 2), (16, 16), (17, 0), (33, 5), (100, 100)])
def test_glue(width, n, commit):
    """A product, at most four sums, an exponential and a division: 12 roundings of terms no larger than |w| |x| + |bias|; the gates likewise."""
    rng = np.random.default_rng(100 * width + n)
    nk, nv, hk, hv = 1, 5, 64, 16
    ch = 2 * nk * hk + nv * hv
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, w, bias, a, b, st = f(n, ch), f(ch, width), f(ch) if n % 2 else None, 4 * f(n, nv), 4 * f(n, nv), f(width - 1, ch)
    a[0, 0], a[0, 1], b[0, 0], b[0, 1] = 60, -60, 100, -100
    a_log, dt_bias = f(nv), f(nv)
    with PooledAttn(CTX, 256, max_cols=100) as pa:
        dn = pa.delta(dict(n_k_heads=nk, n_v_heads=nv, head_k=hk, head_v=hv, conv_width=width, n_layers=2))
        if width > 1:
            pa.delta_write(dn, 1, 1, st)
        y, g, beta = _glue(pa, dn, 1, x, w, bias, a, b, a_log, dt_bias, commit, 4 * (n % 2))
        ry, rg, rbeta, rst = B.delta_glue(x, w, bias, a, b, a_log, dt_bias, st, commit=commit)
        if width > 1:
            assert np.array_equal(pa.delta_read(dn, 1, 1).reshape(st.shape), rst.astype(np.float32)), "the convolution's inputs are copies"
            assert not np.any(pa.delta_read(dn, 0, 1)), "the other layer's state was touched"
    line = np.abs(np.concatenate([st, x])).astype(np.float64)
    size = sum(line[j:j + n] * np.abs(w[:, j]) for j in range(width)) + (0 if bias is None else np.abs(bias))
    assert np.all(np.abs(y - ry) <= 12 * 2.0 ** -24 * 1.1 * size + 1e-30)                        # |silu'| <= 1.1
    assert np.all(np.abs(g - rg) <= 12 * 2.0 ** -24 * (np.abs(rg) + np.exp(a_log) * np.abs(a + dt_bias) * B.sigmoid(a + dt_bias)) + 1e-37)
    assert np.all(np.abs(beta - rbeta) <= 12 * 2.0 ** -24 * rbeta * (1 + np.abs(b) * (1 - rbeta)) + 1e-37)


def test_glue_in_pieces_has_the_bits_of_one_call():
    rng = np.random.default_rng(17)
    nk, nv, hk, hv, n = 1, 2, 64, 32, 40
    ch = 2 * nk * hk + nv * hv
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, w, bias, a, b, a_log, dt_bias = f(n, ch), f(ch, 4), f(ch), f(n, nv), f(n, nv), f(nv), f(nv)
    with PooledAttn(CTX, 256, max_cols=64) as pa:
        dn = pa.delta(dict(n_k_heads=nk, n_v_heads=nv, head_k=hk, head_v=hv, conv_width=4, n_layers=2))
        whole = _glue(pa, dn, 0, x, w, bias, a, b, a_log, dt_bias, n, 0)
        parts = [_glue(pa, dn, 1, x[i:j], w, bias, a[i:j], b[i:j], a_log, dt_bias, j - i, 0) for i, j in ((0, 1), (1, 2), (2, 4), (4, 23), (23, 40))]
        for m in range(3):
            assert np.array_equal(bits(whole[m]), bits(np.concatenate([p[m] for p in parts])))
        assert np.array_equal(pa.delta_read(dn, 0, 1), pa.delta_read(dn, 1, 1))
        pa.delta_reset(dn, 0)
        assert not np.any(pa.delta_read(dn, 0, 1)) and not np.any(pa.delta_read(dn, 0, 0)) and np.any(pa.delta_read(dn, 1, 1))


# ---- handles and refusals ---------------------------------------------------------------------------------------------

def test_create_refusals():
    good = dict(n_k_heads=2, n_v_heads=4, head_k=128, head_v=128, conv_width=4)
    with PooledAttn(CTX, 32, max_cols=16) as pa:
        for bad, code in ((dict(n_k_heads=0), PA_ERR_INVALID), (dict(n_v_heads=3), PA_ERR_INVALID), (dict(n_v_heads=0), PA_ERR_INVALID), (dict(head_k=96), PA_ERR_UNSUPPORTED),
                          (dict(head_k=256), PA_ERR_UNSUPPORTED), (dict(head_v=24), PA_ERR_UNSUPPORTED), (dict(head_v=0), PA_ERR_UNSUPPORTED), (dict(head_v=528), PA_ERR_UNSUPPORTED),
                          (dict(conv_width=5), PA_ERR_UNSUPPORTED), (dict(n_layers=0), PA_ERR_INVALID), (dict(scale=float("nan")), PA_ERR_INVALID), (dict(eps=-1.0), PA_ERR_INVALID),
                          (dict(eps=float("inf")), PA_ERR_INVALID)):
            with pytest.raises(PaError) as e:
                pa.delta(dict(good, **bad))
            assert e.value.code == code and "pa_delta_create" in str(e.value), (bad, str(e.value))
        c = capi.PaDeltaConfig(2, 4, 128, 128, 0, 1, 0.0, 1e-6, 8)
        h = ctypes.c_void_p()
        assert pa.L.pa_delta_create(pa.ctx, ctypes.byref(c), ctypes.byref(h)) == PA_ERR_INVALID and not h.value


def test_call_refusals():
    c = Case(4, nk=1, nv=2, hk=64, hv=32, pad=0)
    with PooledAttn(CTX, 32, max_cols=4) as pa, PooledAttn(CTX, 32, max_cols=4) as other:
        dn = c.handle(pa)
        c.upload(pa)
        out = pa.alloc(4 * 64 * 4)
        big = pa.alloc(1 << 16)
        ok = dict(layer=0, q=c.dq, qs=64, k=c.dk, ks=64, v=c.dv, vs=64, g=c.dg, b=c.dbeta, gs=2, n=4, commit=4, out=out, os=64, dt=PA_OUT_F32)

        def run(who=pa, **kw):
            a = dict(ok, **kw)
            who.delta_decode(dn, a["layer"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["g"], a["b"], a["gs"], a["n"], a["commit"], a["out"], a["os"], a["dt"])
        run()

        class Null:
            ptr = None
        state = Part(out, 0)
        state.ptr = pa.delta_state_ptr(dn, 0, 0)
        for bad in (dict(layer=1), dict(n=0, commit=0), dict(n=5), dict(commit=5), dict(qs=60), dict(ks=66), dict(ks=60), dict(vs=63), dict(gs=1), dict(os=63), dict(dt=2), dict(q=Null, out=out),
                    dict(k=Null), dict(v=Null), dict(g=Null), dict(b=Null), dict(out=None, commit=0), dict(k=Part(big, 4)), dict(q=Part(big, 8)), dict(v=Part(big, 2)), dict(out=Part(big, 1)),
                    dict(out=c.dv), dict(out=c.dq), dict(out=c.dk), dict(out=Part(c.dv, 4 * 63)), dict(out=c.dg), dict(out=state)):
            with pytest.raises(PaError) as e:
                run(**bad)
            assert e.value.code == PA_ERR_INVALID and "pa_delta_decode" in str(e.value), (bad, str(e.value))
        with pytest.raises(PaError) as e:
            run(who=other)
        assert e.value.code == PA_ERR_INVALID and "another context" in str(e.value)
        assert other.L.pa_delta_destroy(other.ctx, dn) == PA_ERR_INVALID
        assert pa.L.pa_delta_decode(None, dn, *([0] * 15)) == PA_ERR_INVALID
        with pytest.raises(PaError) as e:                           # a handle without a convolution
            pa.delta_glue(dn, 0, big, 192, big, None, big, big, 2, big, big, 1, 1, out, 192, out, out, 2)
        assert e.value.code == PA_ERR_INVALID and "without a convolution" in str(e.value)
        assert pa.L.pa_delta_state_bytes(dn, 1) == 0 and pa.delta_state_ptr(dn, 0, 1) is None and pa.delta_state_ptr(dn, 1, 0) is None
        with pytest.raises(PaError):
            pa._chk(pa.L.pa_delta_read(pa.ctx, dn, 0, 1, big.ptr))
        pa.delta_destroy(dn)


def test_glue_refusals():
    with PooledAttn(CTX, 32, max_cols=4) as pa:
        dn = pa.delta(dict(n_k_heads=1, n_v_heads=2, head_k=64, head_v=32, conv_width=4))
        x, w, b, a, small = (pa.alloc(8192) for _ in range(5))
        out, g, beta = (pa.alloc(8192) for _ in range(3))
        ok = dict(x=x, xs=192, w=w, b=b, a=a, bb=a, s=2, al=small, dt=small, n=4, commit=4, out=out, os=192, g=g, beta=beta, gs=2)

        def run(**kw):
            d = dict(ok, **kw)
            pa.delta_glue(dn, 0, d["x"], d["xs"], d["w"], d["b"], d["a"], d["bb"], d["s"], d["al"], d["dt"], d["n"], d["commit"], d["out"], d["os"], d["g"], d["beta"], d["gs"])
        run(); run(b=None)

        class Null:
            ptr = None
        for bad in (dict(n=0, commit=0), dict(n=5), dict(commit=5), dict(xs=188), dict(xs=194), dict(os=190), dict(s=1), dict(gs=1), dict(x=Part(x, 4)), dict(w=Part(w, 8)), dict(b=Part(b, 4)),
                    dict(out=Part(out, 4)), dict(out=x), dict(out=w), dict(g=a), dict(beta=Part(x, 16)), dict(x=Null), dict(w=Null), dict(a=Null), dict(bb=Null), dict(al=Null), dict(dt=Null),
                    dict(out=Null), dict(g=Null), dict(beta=Null), dict(a=Part(a, 2))):
            with pytest.raises(PaError) as e:
                run(**bad)
            assert e.value.code == PA_ERR_INVALID and "pa_delta_glue" in str(e.value), (bad, str(e.value))
