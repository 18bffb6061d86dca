"""The mixture-of-experts layer through the C ABI against the 64-bit oracle.

Tolerance, relative to the 2-norm of what the layer adds to the residual.  A dot product of the layer is per lane at most 32 products one after another per block, the lane's blocks one
after another (dim <= 8192: 4, ffn x slots <= 8192: 4) and 6 levels over the lanes: at most 48 roundings of 2^-24 on a path; three such products, the norm, an exponential, a division and
the weighting lie between x and y: at most 4 x 48 roundings, independent of one another, of terms whose sum of squares is at most that of the products: RTOL = 4 x 48 x 2^-24 = 1.1e-5.  y itself is rounded once more."""
import ctypes

import numpy as np
import pytest
from oracle import blocks_oracle as B
from pooled_amd import capi
from pooled_amd.capi import PooledAttn, PaError, PA_ERR_INVALID, PA_ERR_UNSUPPORTED, PA_W_F32, PA_W_Q4_0, PA_W_Q8_0

pytestmark = pytest.mark.gpu
CTX = dict(n_heads=1, n_kv_heads=1, head_dim=128, n_rot=64, rope_theta=1e6, eps=1e-6)
RTOL = 4 * 48 * 2.0 ** -24


def planes(rng, kind, n, rows, cols):
    lead = (n,) if n else ()
    if kind == PA_W_F32:
        return (rng.standard_normal(lead + (rows, cols)) / cols ** 0.5).astype(np.float32), None
    s = rng.uniform(0.5, 1.5, lead + (rows, cols // 32))
    if kind == PA_W_Q8_0:
        return rng.integers(-128, 128, lead + (rows, cols), dtype=np.int8), (s / (73 * cols ** 0.5)).astype(np.float16).view(np.uint16)
    return rng.integers(0, 256, lead + (rows, cols // 2), dtype=np.uint8), (s / (4.5 * cols ** 0.5)).astype(np.float16).view(np.uint16)


def experts(rng, kind, n, dim, ffn):
    d = {}
    for name, rows, cols in (("gate", ffn, dim), ("up", ffn, dim), ("down", dim, ffn)):
        d[name], d[name + "_s"] = planes(rng, kind, n, rows, cols)
    return d


class Layer:
    def __init__(self, dim=256, ffn=96, E=12, top_k=3, kind=PA_W_Q4_0, shared=True, renorm=True, seed=0):
        rng = np.random.default_rng(seed)
        self.dim, self.ffn, self.E, self.top_k, self.kind, self.renorm = dim, ffn, E, top_k, kind, renorm
        self.router = (rng.standard_normal((E, dim)) * 1.5 / dim ** 0.5).astype(np.float32)
        self.ex = experts(rng, kind, E, dim, ffn)
        self.shared = dict(experts(rng, kind, 0, dim, ffn), weight=(rng.standard_normal(dim) / dim ** 0.5).astype(np.float32)) if shared else None
        self.norm = (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)
        self.rng = rng

    def handle(self, pa):
        return pa.moe(dict(dim=self.dim, ffn=self.ffn, n_experts=self.E, top_k=self.top_k, kind=self.kind, norm_topk=self.renorm), self.router, self.ex, self.shared)

    def oracle(self, x, norm=True):
        return B.moe_layer(x, self.norm if norm else None, self.router, self.ex, self.top_k, self.kind, self.renorm, self.shared)

    def call(self, pa, h, x, norm=True, in_place=False, choice=True, pad=4):
        n, dim = x.shape
        wide = np.concatenate([x, np.full((n, pad), np.nan, np.float32)], 1)
        dx = pa.to_device(wide)
        dy = dx if in_place else pa.to_device(np.full((n + 1, dim + 2 * pad), 777.0, np.float32))
        ids, w = (pa.to_device(np.zeros((n + 1, self.top_k), np.uint32)), pa.to_device(np.zeros((n + 1, self.top_k), np.float32))) if choice else (None, None)
        pa.moe_layer(h, pa.to_device(self.norm) if norm else None, dx, dim + pad, n, dy, dim + (pad if in_place else 2 * pad), ids, w)
        pa.sync()
        if in_place:
            y = dy.download(np.float32, n * (dim + pad)).reshape(n, dim + pad)
            assert np.all(np.isnan(y[:, dim:])) or not pad
            y = y[:, :dim]
        else:
            y = dy.download(np.float32, (n + 1) * (dim + 2 * pad)).reshape(n + 1, dim + 2 * pad)
            assert np.all(y[n] == 777.0) and np.all(y[:n, dim:] == 777.0), "wrote outside the columns"
            y = y[:n, :dim]
        if not choice:
            return y, None, None
        i, ww = ids.download(np.uint32, (n + 1) * self.top_k).reshape(n + 1, -1), w.download(np.float32, (n + 1) * self.top_k).reshape(n + 1, -1)
        assert not i[n].any() and not ww[n].any(), "wrote outside the choices"
        return y, i[:n], ww[:n]


def close(y, x, ref, what=""):
    added, got = ref - x, y.astype(np.float64) - x
    assert np.all(np.isfinite(y))
    d = np.sqrt(((got - added) ** 2).sum(-1)) / np.sqrt((added ** 2).sum(-1))
    room = RTOL + 2.0 ** -24 * np.sqrt((ref ** 2).sum(-1) / (added ** 2).sum(-1))
    print("%s relative error %.2e of %.2e" % (what, d.max(), room.max()))
    assert np.all(d <= room), (what, d.max(), room)


KINDS = {"f32": PA_W_F32, "q8_0": PA_W_Q8_0, "q4_0": PA_W_Q4_0}
SIZES = [dict(dim=256, ffn=96, E=12, top_k=3), dict(dim=32, ffn=32, E=1, top_k=1), dict(dim=2048, ffn=512, E=20, top_k=8), dict(dim=1056, ffn=352, E=61, top_k=5),
         dict(dim=2080, ffn=2144, E=3, top_k=2), dict(dim=64, ffn=160, E=300, top_k=16), dict(dim=4128, ffn=32, E=5, top_k=5)]


@pytest.mark.parametrize("n", [1, 2, 5, 16, 33])
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_layer(size, kind, n):
    if SIZES[size]["dim"] > 2000 and n == 33:
        n = 3
    L = Layer(kind=KINDS[kind], shared=(size + n) % 2 == 0, renorm=n % 3 != 0, seed=7 * size + n, **SIZES[size])
    x = (L.rng.standard_normal((n, L.dim)) * 2).astype(np.float32)
    with PooledAttn(CTX, 64, max_cols=max(n, 2)) as pa:
        h = L.handle(pa)
        y, ids, w = L.call(pa, h, x, in_place=n == 2, pad=0 if n == 5 else 4)
        ref, rids, rw = L.oracle(x)
        assert np.array_equal(ids, rids), "other experts than the oracle's"
        assert np.all(np.abs(w - rw) <= RTOL * rw * 20)              # |d p / p| <= 2 |d logit|, logits of a few units
        close(y, x, ref, "y")


def test_without_norm_and_without_choice():
    L = Layer(seed=3)
    x = L.rng.standard_normal((3, L.dim)).astype(np.float32)
    with PooledAttn(CTX, 64, max_cols=4) as pa:
        y, _, _ = L.call(pa, L.handle(pa), x, norm=False, choice=False)
        close(y, x, L.oracle(x, norm=False)[0])


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_a_token_has_its_bits_in_every_company(kind):
    L = Layer(dim=512, ffn=160, E=9, top_k=4, kind=KINDS[kind], seed=4)
    x = L.rng.standard_normal((37, L.dim)).astype(np.float32)
    x[5] = x[11]                                                   # the same token twice
    with PooledAttn(CTX, 64, max_cols=40) as pa:
        h = L.handle(pa)
        whole = L.call(pa, h, x)
        again = L.call(pa, h, x, in_place=True)
        for a, b in zip(whole, again):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32)), "two calls differ"
        for c0, c1 in ((0, 1), (1, 3), (3, 8), (8, 37), (11, 12), (36, 37)):
            part = L.call(pa, h, x[c0:c1])
            for a, b in zip(whole, part):
                assert np.array_equal(a[c0:c1].view(np.uint32), b.view(np.uint32)), "columns %d .. %d depend on their company" % (c0, c1)
        assert np.array_equal(whole[0][5], whole[0][11])


def test_equal_logits_go_to_the_lowest_index():
    L = Layer(dim=64, ffn=32, E=130, top_k=6, kind=PA_W_F32, shared=False, seed=5)
    L.router[:] = 0
    L.router[[7, 70, 128]] = L.rng.standard_normal(64).astype(np.float32)
    x = L.rng.standard_normal((8, 64)).astype(np.float32)
    with PooledAttn(CTX, 64, max_cols=8) as pa:
        y, ids, w = L.call(pa, L.handle(pa), x)
    ref, rids, rw = L.oracle(x)
    up = (x / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True)) * L.norm) @ L.router[7] > 0
    for t in range(8):
        assert ids[t].tolist() == ([7, 70, 128, 0, 1, 2] if up[t] else [0, 1, 2, 3, 4, 5])
    close(y, x, ref)


def test_all_tokens_on_one_expert():
    L = Layer(dim=256, ffn=64, E=40, top_k=1, kind=PA_W_Q8_0, seed=6)
    x = np.abs(L.rng.standard_normal((32, 256))).astype(np.float32)
    L.router[17] = 1
    with PooledAttn(CTX, 64, max_cols=32) as pa:
        y, ids, w = L.call(pa, L.handle(pa), x)
    assert np.all(ids == 17) and np.all(w == 1)
    close(y, x, L.oracle(x)[0])


@pytest.mark.parametrize("renorm", [True, False])
def test_nan_and_infinity_stay_with_their_token(renorm):
    L = Layer(dim=128, ffn=64, E=70, top_k=4, seed=8, renorm=renorm)
    x = L.rng.standard_normal((6, 128)).astype(np.float32)
    clean = x.copy()
    x[1, 3], x[4, 100] = np.nan, np.inf
    with PooledAttn(CTX, 64, max_cols=8) as pa:
        h = L.handle(pa)
        y, ids, w = L.call(pa, h, x)
        want = L.call(pa, h, clean)
    for t in range(6):
        if t in (1, 4):
            assert np.all(np.isnan(y[t])) and np.all(np.isnan(w[t])) and np.all(ids[t] < 70) and len(set(ids[t])) == 4
        else:
            assert np.array_equal(y[t], want[0][t]) and np.array_equal(ids[t], want[1][t])


def test_logits_far_apart():
    L = Layer(dim=64, ffn=32, E=10, top_k=10, kind=PA_W_F32, seed=9, renorm=False)
    L.router *= 300                                                # most probabilities underflow
    x = L.rng.standard_normal((5, 64)).astype(np.float32)
    with PooledAttn(CTX, 64, max_cols=8) as pa:
        y, ids, w = L.call(pa, L.handle(pa), x)
    ref, rids, rw = L.oracle(x)
    assert np.array_equal(ids, rids) and np.all(np.isfinite(w)) and np.all(np.abs(w - rw) <= 64 * 2.0 ** -24 * 2000)     # an error of 2^-24 of a logit of some 2000
    close(y, x, x + (ref - x))


def test_create_refusals():
    rng = np.random.default_rng(0)
    with PooledAttn(CTX, 32, max_cols=4) as pa:
        def make(dim=64, ffn=32, n_experts=4, top_k=2, kind=PA_W_Q4_0, flags=0, null=(), shared_null=()):
            c = capi.PaMoeConfig(dim, ffn, n_experts, top_k, kind, flags)
            buf = rng.integers(0, 255, 1 << 16, dtype=np.uint8)
            pl = capi.PaMoePlanes(**{n: None if n in null else buf.ctypes.data for n, _ in capi.PaMoePlanes._fields_})
            h = ctypes.c_void_p()
            rc = pa.L.pa_moe_create(pa.ctx, ctypes.byref(c), ctypes.byref(pl), ctypes.byref(h))
            if rc == 0:
                pa.L.pa_moe_destroy(pa.ctx, h)
            else:
                assert not h.value and "pa_moe_create" in pa.L.pa_last_error(pa.ctx).decode()
            return rc
        assert make() == 0 and make(flags=3) == 0
        assert make(kind=PA_W_F32, null=("h_gate_s", "h_up_s", "h_down_s", "h_shared_gate_s", "h_shared_up_s", "h_shared_down_s"), flags=2) == 0
        for bad in (dict(dim=0), dict(dim=48), dict(ffn=0), dict(ffn=33), dict(n_experts=0), dict(top_k=0), dict(top_k=5), dict(kind=3), dict(kind=-1), dict(flags=4), dict(null=("h_router",)),
                    dict(null=("h_gate",)), dict(null=("h_up_s",)), dict(null=("h_down",)), dict(flags=2, null=("h_shared_gate",)), dict(flags=2, null=("h_shared_down_w",)),
                    dict(flags=2, null=("h_shared_up_s",))):
            assert make(**bad) == PA_ERR_INVALID, bad
        for bad in (dict(dim=8224), dict(ffn=8224), dict(n_experts=1025), dict(n_experts=32, top_k=17)):
            assert make(**bad) == PA_ERR_UNSUPPORTED, bad


def test_call_refusals():
    L = Layer(dim=64, ffn=32, E=4, top_k=2, seed=1)
    with PooledAttn(CTX, 32, max_cols=4) as pa, PooledAttn(CTX, 32, max_cols=4) as other:
        h = L.handle(pa)
        x, y, nw, ids, w = (pa.to_device(np.zeros(512, np.float32)) for _ in range(5))
        ok = dict(nw=nw, x=x, xs=64, n=4, y=y, ys=64, ids=ids, w=w)

        class Null:
            ptr = None

        def part(b, at):
            p = type("P", (), {})()
            p.ptr = b.ptr + at
            return p

        def run(who=pa, **kw):
            a = dict(ok, **kw)
            who.moe_layer(h, a["nw"], a["x"], a["xs"], a["n"], a["y"], a["ys"], a["ids"], a["w"])
        run(); run(y=x); run(nw=None, ids=None, w=None)
        for bad in (dict(x=Null), dict(y=Null), dict(n=0), dict(n=5), dict(xs=60), dict(xs=66), dict(ys=60), dict(ys=65), dict(x=part(x, 4)), dict(y=part(y, 8)), dict(nw=part(nw, 4)),
                    dict(ids=part(ids, 2)), dict(w=part(w, 1)), dict(y=part(x, 16)), dict(y=x, ys=68), dict(y=nw), dict(ids=x), dict(w=y), dict(w=ids), dict(ids=nw)):
            with pytest.raises(PaError) as e:
                run(**bad)
            assert e.value.code == PA_ERR_INVALID and "pa_moe_layer" in str(e.value), (bad, str(e.value))
        with pytest.raises(PaError) as e:
            run(who=other)
        assert "another context" in str(e.value)
        assert other.L.pa_moe_destroy(other.ctx, h) == PA_ERR_INVALID
        assert pa.L.pa_moe_layer(None, h, *([0] * 8)) == PA_ERR_INVALID
