"""The mixture-of-experts layer where one value is far larger than those beside it, against the 64-bit oracle.  Tolerance: test_gpu_moe's, RTOL of the 2-norm of what the layer adds."""
import numpy as np
import pytest
from oracle import blocks_oracle as B
from pooled_amd.capi import PooledAttn, PA_W_Q4_0, PA_W_Q8_0
from test_gpu_moe import CTX, RTOL, Layer

pytestmark = pytest.mark.gpu


def no_weight(L, name, at):
    """Element `at` of every row of the planes `name` is a weight of zero."""
    for d in [L.ex] + ([L.shared] if L.shared else []):
        if L.kind == PA_W_Q8_0:
            d[name][..., at] = 0
        else:                                          # a block's byte j holds elements j (low) and j + 16 (high); 8 stands for zero
            byte = d[name][..., at // 32 * 16 + at % 16]
            d[name][..., at // 32 * 16 + at % 16] = (byte & 0x0F) | 0x80 if at % 32 >= 16 else (byte & 0xF0) | 0x08


def check(L, x, rows, norm=False):
    with PooledAttn(CTX, 64, max_cols=max(len(x), 2)) as pa:
        y, ids, _ = L.call(pa, L.handle(pa), x, norm=norm)
    ref, rids, _ = L.oracle(x, norm=norm)
    assert np.array_equal(ids, rids)
    added, got = (ref - x)[:, rows], (y.astype(np.float64) - x)[:, rows]
    d = np.sqrt(((got - added) ** 2).sum(-1) / (added ** 2).sum(-1))
    room = RTOL + 2.0 ** -24 * np.sqrt((ref[:, rows] ** 2).sum(-1) / (added ** 2).sum(-1))
    print("relative error %.2e of %.2e" % (d.max(), room.min()))
    assert np.all(d <= room)


@pytest.mark.parametrize("n", [1, 3, 20])
@pytest.mark.parametrize("at", [5, 90])
@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e6])
@pytest.mark.parametrize("kind", [PA_W_Q4_0, PA_W_Q8_0])
def test_a_large_activation_without_weight(kind, ratio, at, n):
    """One channel of the residual is `ratio` times the others and no expert looks at it: gate, up and what follows are as exact as without it."""
    L = Layer(dim=256, ffn=96, E=12, top_k=3, kind=kind, seed=int(np.log10(ratio)) + at)
    for name in ("gate", "up"):
        no_weight(L, name, at)
    L.router[:, at] = 0; L.shared["weight"][at] = 0
    x = L.rng.standard_normal((n, L.dim)).astype(np.float32)
    x[:, at] = ratio * (1 + 0.1 * L.rng.random(n))
    check(L, x, np.arange(L.dim) != at)


@pytest.mark.parametrize("n", [1, 3, 20])
@pytest.mark.parametrize("at", [3, 84])
@pytest.mark.parametrize("kind", [PA_W_Q4_0, PA_W_Q8_0])
def test_a_large_expert_value_without_weight(kind, at, n):
    """One value of an expert's hidden layer is some 1e6 times the others and has no weight in the projection down."""
    L = Layer(dim=256, ffn=96, E=12, top_k=3, kind=kind, seed=at + n)
    for d in (L.ex, L.shared):
        for name in ("gate_s", "up_s"):
            s = d[name].view(np.float16)
            s[..., at, :] = (s[..., at, :].astype(np.float32) * 1000).astype(np.float16)
    no_weight(L, "down", at)
    x = L.rng.standard_normal((n, L.dim)).astype(np.float32)
    check(L, x, slice(None))


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("size,eps", [(1e15, 1e-6), (1e19, 1e-6), (1e25, 1e-6), (1e37, 1e-6), (1e-12, 0.0), (1e-20, 0.0), (1e-30, 0.0)])
def test_residuals_whose_squares_leave_f32(size, eps, n):
    """The norm takes the size out: choices, weights and what is added are those of a residual of ordinary size."""
    L = Layer(dim=1056, ffn=64, E=12, top_k=3, kind=PA_W_Q4_0, seed=int(abs(np.log10(size))))
    x = (L.rng.standard_normal((n, L.dim)) * size).astype(np.float32)
    with PooledAttn(dict(CTX, eps=eps), 64, max_cols=max(n, 2)) as pa:
        y, ids, w = L.call(pa, L.handle(pa), x)
    ref, rids, rw = B.moe_layer(x, L.norm, L.router, L.ex, L.top_k, L.kind, L.renorm, L.shared, eps=eps)
    assert np.array_equal(ids, rids)
    assert np.all(np.abs(w - rw) <= RTOL * rw * 20)                  # as in test_gpu_moe
    # test_gpu_moe's condition times the norm of what is added: that is nothing in 64 bits beside the largest residuals
    d = np.sqrt(((y.astype(np.float64) - ref) ** 2).sum(-1))
    room = RTOL * np.sqrt(((ref - x) ** 2).sum(-1)) + 2.0 ** -24 * np.sqrt((ref ** 2).sum(-1))
    print("error %.2e of %.2e" % (d.max(), room.min()))
    assert np.all(d <= room)
