"""The delta rule, its pre-step and the experts run together as a model runs them: a layer of one-token steps and of a prompt against the 64-bit oracle, a recorded step
replayed from a HIP graph, and calls on a stream that the caller chose.

Tolerance of a layer, relative to what it adds to the residual of a token: the roundings on a path from its input to its output are at most 24 of each projection, 12 of the
pre-step, 24 (1 + sqrt(n)) of the rule after n tokens (eight times that in chunks) and 192 of the experts, and a stage passes on at most 4 times the relative error of its input
(a division by a norm, silu, softmax of logits of a size below 4)."""
import ctypes

import numpy as np
import pytest
from oracle import blocks_oracle as B
from pooled_amd.capi import PooledAttn, PA_W_F32, PA_W_Q4_0, PA_W_Q8_0
from test_gpu_delta import Part
from test_gpu_graph import _hip, _ok
from test_gpu_moe import experts

pytestmark = pytest.mark.gpu
vp = ctypes.c_void_p
CTX = dict(n_heads=1, n_kv_heads=1, head_dim=128, n_rot=64, rope_theta=1e6, eps=1e-6)
DIM, FFN, E, TOP = 256, 96, 24, 4
NK, NV, HK, HV, W = 2, 4, 64, 32, 4
KEY, VAL = NK * HK, NV * HV
CH = 2 * KEY + VAL


def tol(n, chunks):
    return 4 * (24 + 12 + 24 * (1 + n ** 0.5) * (8 if chunks else 1) + 24 + 192) * 2.0 ** -24


class Model:
    """x += w_o rule(pre-step(w_in rmsnorm(x)));  x += experts(rmsnorm(x))"""

    def __init__(self, kind, seed):
        rng = self.rng = np.random.default_rng(seed)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.kind = kind
        self.w_in, self.w_o = f(CH + 2 * NV, DIM) / 16, f(DIM, VAL) / 2
        self.norm1, self.norm2 = 1 + 0.1 * f(DIM), 1 + 0.1 * f(DIM)
        self.conv, self.bias, self.a_log, self.dt = f(CH, W) / 2, 0.1 * f(CH), f(NV), f(NV)
        self.router = 2 * f(E, DIM) / 16
        self.ex = experts(rng, kind, E, DIM, FFN)
        self.shared = dict(experts(rng, kind, 0, DIM, FFN), weight=f(DIM) / 16)

    def oracle(self, x):
        """the residuals behind the rule and behind the experts, the projected columns, the choices and the states"""
        x = x.astype(np.float64)
        xn = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + 1e-6) * self.norm1
        y = xn @ self.w_in.astype(np.float64).T
        c, g, beta, conv = B.delta_glue(y[:, :CH], self.conv, self.bias, y[:, CH:CH + NV], y[:, CH + NV:], self.a_log, self.dt, np.zeros((W - 1, CH)))
        n = len(x)
        o, S = B.delta_rule(c[:, :KEY].reshape(n, NK, HK), c[:, KEY:2 * KEY].reshape(n, NK, HK), c[:, 2 * KEY:].reshape(n, NV, HV), g, beta, np.zeros((NV, HV, HK)))
        mid = x + o.reshape(n, VAL) @ self.w_o.astype(np.float64).T
        out, ids, _ = B.moe_layer(mid, self.norm2, self.router, self.ex, TOP, self.kind, True, self.shared)
        return mid, out, y, ids, S, conv

    def device(self, pa):
        up = pa.to_device
        self.d = dict(norm1=up(self.norm1), norm2=up(self.norm2), conv=up(self.conv), bias=up(self.bias), a_log=up(self.a_log), dt=up(self.dt))
        self.h_in, self.h_o = pa.weight(PA_W_F32, self.w_in), pa.weight(PA_W_F32, self.w_o)
        self.dn = pa.delta(dict(n_k_heads=NK, n_v_heads=NV, head_k=HK, head_v=HV, conv_width=W))
        self.moe = pa.moe(dict(dim=DIM, ffn=FFN, n_experts=E, top_k=TOP, kind=self.kind, norm_topk=True), self.router, self.ex, self.shared)
        return self

    def rule(self, pa, y, n, call, out):
        """n projected columns y [n][CH + 2 NV] through pre-step and rule"""
        d, st = self.d, CH + 2 * NV
        if not hasattr(self, "c") or self.c[2] < n:
            self.c = (pa.alloc(n * CH * 4), pa.alloc(2 * n * NV * 4), n)
        c, gates = self.c[0], self.c[1]
        g, beta = gates, Part(gates, n * NV * 4)
        pa.delta_glue(self.dn, 0, y, st, d["conv"], d["bias"], Part(y, CH * 4), Part(y, (CH + NV) * 4), st, d["a_log"], d["dt"], n, n, c, CH, g, beta, NV)
        q, k, v = c, Part(c, KEY * 4), Part(c, 2 * KEY * 4)
        if call == "decode":
            pa.delta_decode(self.dn, 0, q, CH, k, CH, v, CH, g, beta, NV, n, n, out, VAL)
        else:
            pa.delta_prefill(self.dn, 0, q, CH, k, CH, v, CH, g, beta, NV, n, out, VAL)

    def step(self, pa, x, y, out):
        """one token, residual x in place"""
        pa.gemv_norm(self.h_in, x, self.d["norm1"], y)
        self.rule(pa, y, 1, "decode", out)
        pa.gemv(self.h_o, out, x, acc=True)
        pa.moe_layer(self.moe, self.d["norm2"], x, DIM, 1, x, DIM)


def close(got, ref, base, room, what):
    d = np.sqrt(((got.astype(np.float64) - ref) ** 2).sum(-1)) / np.sqrt(((ref - base) ** 2).sum(-1))
    room = room + 2.0 ** -23 * np.sqrt((ref ** 2).sum(-1) / ((ref - base) ** 2).sum(-1))
    print("%s: %.2e of %.2e" % (what, d.max(), room.max()))
    assert np.all(d <= room), (what, d.max())


@pytest.mark.parametrize("kind", [PA_W_F32, PA_W_Q8_0, PA_W_Q4_0])
def test_tokens_through_a_layer(kind):
    m = Model(kind, 3 + kind)
    n = 6
    x = m.rng.standard_normal((n, DIM)).astype(np.float32)
    mid, ref, _, _, S, conv = m.oracle(x)
    with PooledAttn(CTX, 64, max_cols=2) as pa:
        m.device(pa)
        dx, y, out = pa.alloc(DIM * 4), pa.alloc((CH + 2 * NV) * 4), pa.alloc(VAL * 4)
        got = []
        for t in range(n):
            dx.upload(x[t])
            m.step(pa, dx, y, out)
            pa.sync()
            got.append(dx.download(np.float32, DIM).copy())
        close(np.array(got), ref, x, tol(n, False), "residual")
        s = pa.delta_read(m.dn, 0, 0).reshape(S.shape)
        assert np.sqrt(((s - S) ** 2).sum()) <= tol(n, False) * np.sqrt((S ** 2).sum())


@pytest.mark.parametrize("n", [47, 64, 150])
def test_a_prompt_then_tokens(n):
    """n columns as a prompt, then two of them as tokens: the same as all of them token by token in the oracle."""
    m = Model(PA_W_Q8_0, 20 + n)
    x = m.rng.standard_normal((n + 2, DIM)).astype(np.float32)
    mid, ref, cols, ids, S, _ = m.oracle(x)
    with PooledAttn(CTX, 256, max_cols=160) as pa:
        m.device(pa)
        y, out = pa.to_device(cols[:n].astype(np.float32)), pa.alloc(n * VAL * 4)
        m.rule(pa, y, n, "prefill", out)
        rows = (mid[:n] - x[:n])
        pa.sync()
        o = out.download(np.float32, n * VAL).reshape(n, VAL).astype(np.float64) @ m.w_o.astype(np.float64).T
        close(o, rows, 0 * rows, tol(n, True), "rule")
        # the experts over all columns at once, from the oracle's residual
        dx = pa.to_device(mid[:n].astype(np.float32)); dids = pa.to_device(np.zeros((n, TOP), np.uint32))
        pa.moe_layer(m.moe, m.d["norm2"], dx, DIM, n, dx, DIM, dids, None)
        pa.sync()
        close(dx.download(np.float32, n * DIM).reshape(n, DIM), ref[:n], mid[:n], tol(1, False), "experts")
        assert np.array_equal(dids.download(np.uint32, n * TOP).reshape(n, TOP), ids[:n])
        x1, y1, o1 = pa.alloc(DIM * 4), pa.alloc((CH + 2 * NV) * 4), pa.alloc(VAL * 4)
        for t in (n, n + 1):
            x1.upload(x[t])
            m.step(pa, x1, y1, o1)
            pa.sync()
            close(x1.download(np.float32, DIM)[None], ref[t:t + 1], x[t:t + 1], tol(n, True), "token %d" % t)


@pytest.mark.parametrize("n", [1, 5, 16, 130])
def test_replayed_from_a_graph(n):
    """Recorded once, replayed three times with eager work on the same handles between: every replay has the bits of the eager run from the same state."""
    m = Model(PA_W_Q4_0, 40 + n)
    x = m.rng.standard_normal((n, DIM)).astype(np.float32)
    cols = m.rng.standard_normal((n, CH + 2 * NV)).astype(np.float32)
    S0 = (0.1 * m.rng.standard_normal(NV * HV * HK)).astype(np.float32)
    conv0 = m.rng.standard_normal((W - 1) * CH).astype(np.float32)
    hip = _hip()
    stream = vp()
    _ok(hip.hipStreamCreate(ctypes.byref(stream)), "hipStreamCreate")
    with PooledAttn(CTX, 256, max_cols=160) as pa:
        pa._chk(pa.L.pa_set_stream(pa.ctx, stream))
        m.device(pa)
        y, out, dx = pa.to_device(cols), pa.alloc(n * VAL * 4), pa.alloc(n * DIM * 4)

        def start():
            pa.delta_write(m.dn, 0, 0, S0); pa.delta_write(m.dn, 0, 1, conv0); dx.upload(x); out.upload(np.full(n * VAL, 777.0, np.float32))

        def sequence():
            m.rule(pa, y, n, "decode" if n <= 16 else "prefill", out)
            pa.moe_layer(m.moe, m.d["norm2"], dx, DIM, n, dx, DIM)

        def results():
            pa.sync()
            return [out.download(np.float32, n * VAL).copy(), dx.download(np.float32, n * DIM).copy(), pa.delta_read(m.dn, 0, 0), pa.delta_read(m.dn, 0, 1)]

        start(); sequence()
        eager = results()
        assert all(np.all(np.isfinite(a)) for a in eager) and not np.any(eager[0] == 777.0)
        pa.delta_reset(m.dn, 0)
        pa.sync()
        graph, gexec = vp(), vp()
        _ok(hip.hipStreamBeginCapture(stream, 0), "hipStreamBeginCapture")
        sequence()
        _ok(hip.hipStreamEndCapture(stream, ctypes.byref(graph)), "hipStreamEndCapture")
        _ok(hip.hipGraphInstantiate(ctypes.byref(gexec), graph, None, None, 0), "hipGraphInstantiate")
        for rep in range(3):
            sequence()                                       # eager, over whatever state there is
            pa.delta_reset(m.dn, 0)
            start()
            _ok(hip.hipGraphLaunch(gexec, stream), "hipGraphLaunch")
            for a, b in zip(results(), eager):
                assert np.array_equal(a.view(np.uint32), b.view(np.uint32)), "replay %d" % rep
        # a second replay goes on from the state of the first, as a second eager call does
        start(); sequence(); sequence()
        twice = results()
        start()
        _ok(hip.hipGraphLaunch(gexec, stream), "hipGraphLaunch"); _ok(hip.hipGraphLaunch(gexec, stream), "hipGraphLaunch")
        for a, b in zip(results(), twice):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
        _ok(hip.hipGraphExecDestroy(gexec), "hipGraphExecDestroy"); _ok(hip.hipGraphDestroy(graph), "hipGraphDestroy")
        pa._chk(pa.L.pa_set_stream(pa.ctx, None))
    _ok(hip.hipStreamDestroy(stream), "hipStreamDestroy")


def test_two_contexts_side_by_side():
    """Two contexts with streams, handles and workspaces of their own, their calls interleaved without waiting: each has the bits that it has alone."""
    n = 90
    hip = _hip()
    alone = []
    models = [Model(PA_W_Q8_0, 70 + i) for i in range(2)]
    data = [(m.rng.standard_normal((n, CH + 2 * NV)).astype(np.float32), m.rng.standard_normal((n, DIM)).astype(np.float32)) for m in models]
    for together in (False, True):
        streams, got = [vp(), vp()], []
        pas = [PooledAttn(CTX, 256, max_cols=160) for _ in models]
        work = []
        for i, (m, pa) in enumerate(zip(models, pas)):
            _ok(hip.hipStreamCreate(ctypes.byref(streams[i])), "hipStreamCreate")
            pa._chk(pa.L.pa_set_stream(pa.ctx, streams[i]))
            m.__dict__.pop("c", None)
            m.device(pa)
            work.append((pa.to_device(data[i][0]), pa.alloc(n * VAL * 4), pa.to_device(data[i][1])))

        def call(i):
            m, pa, (y, out, dx) = models[i], pas[i], work[i]
            m.rule(pa, y, n, "prefill", out)
            pa.moe_layer(m.moe, m.d["norm2"], dx, DIM, n, dx, DIM)
        for i in range(2):
            call(i)                                          # allocates the test's own buffers
        for pa in pas:
            pa.sync()
        for rep in range(5):
            for i in range(2):
                call(i)
                if not together:
                    pas[i].sync()
        for i in range(2):
            pas[i].sync()
            got += [work[i][1].download(np.float32, n * VAL).copy(), work[i][2].download(np.float32, n * DIM).copy(), pas[i].delta_read(models[i].dn, 0, 0)]
        for i, pa in enumerate(pas):
            pa._chk(pa.L.pa_set_stream(pa.ctx, None))
            pa.close()
            _ok(hip.hipStreamDestroy(streams[i]), "hipStreamDestroy")
        alone.append(got)
    for a, b in zip(*alone):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
