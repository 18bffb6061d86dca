"""pa_delta_prefill where sizes change with time: every token is held to f32 rounding of what it takes in, however large or small the tokens around it.

What token t takes in, per value column: M_t = exp(g_t) M_(t-1) + beta_t |v_t|, M_0 the 2-norm of the column's row of the state.  Every quantity of the token is at most a small multiple of
it, and M_i exp(G_t - G_i) <= M_t, so an error of token i arrives as a part of M_t of no more than its own part of M_i.

Tolerances, relative to M_t (2-norm over the value columns of a head).  f32 arithmetic: 24 roundings of 2^-24 on a path (see test_gpu_delta), independent of one another and from token to token:
sqrt(24) 2^-24 (1 + sqrt(n)).  A product of two pairs of f16 (22 bits each) is off by 2 x 2^-23 + 2^-22 = 2^-21, and at most three of them follow one another: 3 x 2^-21 < 2^-19.4.
Halves of a pair have a smallest step: 2^-24 / 2048, half of it 2^-36.  A column's X is scaled to a bound B in [2^13, 2^14), so it is off by 2^-49 B; P, T and P', at most one or two in size
and stored times 2^14, by 2^-50.  Over the 64 tokens of a chunk, independently: sqrt(64) (3 x 2^-50 + 2^-49) B = 40 x 2^-50 B, and a chunk is taken so only if M >= 2^-23 B, as sums over the 32
columns of a workgroup at most, whose 2-norm is no less than 1 / sqrt(32) of them: sqrt(32) x 40 x 2^-27 < 2^-19.1.  Together below 2^-18: TOKEN(n) = sqrt(24) 2^-24 (1 + sqrt(n)) + 2^-18.
A row of the state has 128 of these errors, of K' (2^-49), of T and of K~ (2^-50 each), and that of X: sqrt(64) (sqrt(128) (2^-49 + 2 x 2^-50) + 2^-49) B < 2^-41.4 B, and M >= 2^-23 B
in the column itself: 2^-18.4, so 2^-17 in place of 2^-18."""
import numpy as np
import pytest
from pooled_amd.capi import PooledAttn
from test_gpu_delta import CTX, Case

pytestmark = pytest.mark.gpu


def token_tol(n, floor=2.0 ** -18):
    return 24 ** 0.5 * 2.0 ** -24 * (1 + n ** 0.5) + floor


def taken(c):
    """M [n, nv, hv]"""
    m, rows = np.sqrt((c.state.astype(np.float64) ** 2).sum(-1)), []
    for t in range(c.n):
        m = np.exp(c.g[t].astype(np.float64))[:, None] * m + np.abs(c.beta[t].astype(np.float64)[:, None] * c.v[t])
        rows.append(m)
    return np.array(rows)


def check_tokens(c, kind="prefill", n_layers=1):
    with PooledAttn(CTX, 512, max_cols=max(c.n, 16)) as pa:
        dn = c.handle(pa)
        pa.delta_write(dn, 0, 0, c.state)
        c.upload(pa)
        out, state = c.call(pa, dn, kind), c.read(pa, dn)
    ref, ref_state = c.oracle()
    m = taken(c)
    size = np.sqrt((m ** 2).sum(-1)) * (c.scale or c.hk ** -0.5)     # |q^| <= 1, times the scale
    d = np.sqrt(((out - ref) ** 2).sum(-1))
    off = np.where(size > 0, d / np.where(size > 0, size, 1), np.where(d > 0, np.inf, 0))
    rows = np.sqrt(((state - ref_state) ** 2).sum(-1)) / np.maximum(m[-1], 1e-300)
    print("tokens %.2e of %.2e, at %d;  rows of the state %.2e of %.2e" % (off.max(), token_tol(c.n), np.unravel_index(off.argmax(), off.shape)[0], rows.max(), token_tol(c.n, 2.0 ** -17)))
    assert np.all(np.isfinite(out)) and np.all(np.isfinite(state))
    assert off.max() <= token_tol(c.n)
    assert rows.max() <= token_tol(c.n, 2.0 ** -17)


@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("place", [32, 64, 100, 129])
@pytest.mark.parametrize("ratio", [1e3, 1e5, 1e6, 1e7, 1e8, 1e9, 1e12])
def test_large_values_that_one_token_forgets(kind, ratio, place):
    """Values `ratio` times as large up to a token whose g = -ln ratio brings the state down to what follows: the old values still count in full."""
    c = Case(150, seed=int(np.log10(ratio)) + place, nk=1, nv=2, hv=32)
    c.v[:place] *= np.float32(ratio)
    c.g[place] = -np.log(ratio)
    check_tokens(c, kind)


@pytest.mark.parametrize("ratio", [1e6, 1e8, 1e10])
def test_large_values_forgotten_over_many_tokens(ratio):
    c = Case(200, seed=3, nk=1, nv=2, hv=32)
    c.v[:40] *= np.float32(ratio)
    c.g[40:90] -= np.float32(np.log(ratio) / 50)
    check_tokens(c)


@pytest.mark.parametrize("fresh", [True, False])
@pytest.mark.parametrize("place", [3, 63, 64, 100])
@pytest.mark.parametrize("ratio", [1e3, 1e6, 1e9, 1e12])
def test_small_values_in_front_of_large_ones(ratio, place, fresh):
    """The tokens in front keep their own accuracy, from an empty state or a small one."""
    c = Case(150, seed=place, nk=1, nv=2, hv=32, state=0.0 if fresh else 0.1 / ratio)
    c.v[:place] /= np.float32(ratio)
    check_tokens(c)


@pytest.mark.parametrize("ratio", [1e5, 1e7, 1e9])
@pytest.mark.parametrize("place", [90, 127, 150, 157])
@pytest.mark.parametrize("columns", [slice(0, 1), slice(0, 16), slice(3, None, 5)])
def test_some_value_columns_forget_more_than_others(ratio, place, columns):
    """Large values in some columns alone, forgotten by a token within a chunk or the last of one: those columns' rows of the state, and all tokens."""
    c = Case(128 + 30, seed=7, nk=1, nv=1, hv=64)
    c.v[:place, :, columns] *= np.float32(ratio)
    c.g[place] = -np.log(ratio)
    check_tokens(c)


@pytest.mark.parametrize("n,last", [(128, 127), (150, 149), (150, 146), (193, 192)])
def test_a_column_that_ends_small_beside_one_that_stays_large(n, last):
    """One column's last tokens are 1e-9 of what it had, with a decay that the next column, ever larger, does not show: its row of the state keeps its own accuracy."""
    c = Case(n, seed=n, nk=1, nv=2, hv=32)
    c.g[last] = -np.log(1e9)
    c.v[last:, :, 1::2] *= np.float32(1e9)
    check_tokens(c)


@pytest.mark.parametrize("lead", [1, 40, 64, 100])
def test_tokens_left_out_in_front(lead):
    """beta = 0 and an empty state: nothing is taken in, and the outputs there are exactly zero."""
    c = Case(150, seed=lead, nk=1, nv=2, hv=32, state=0.0)
    c.beta[:lead] = 0
    check_tokens(c)


@pytest.mark.parametrize("hk,nv,hv", [(64, 2, 16), (128, 36, 128), (64, 36, 128)])
def test_sizes_apart_in_every_tile_of_value_columns(hk, nv, hv):
    """16 and 32 value columns a workgroup, both head sizes; some heads forget 1e8, some nothing."""
    c = Case(140, seed=hk + nv, nk=nv // 2, nv=nv, hk=hk, hv=hv)
    c.v[:70, ::2] *= np.float32(1e8)
    c.g[70, ::2] = -np.log(1e8)
    check_tokens(c)


@pytest.mark.parametrize("n", [130, 1000, 2200])
def test_ordinary_tokens_are_as_exact_as_f32(n):
    """Relative to the 2-norm of a head's outputs, as in test_gpu_delta, but roundings count only as long as the state remembers them: sqrt(sum over i of exp(2 (G_t - G_i))) in place of sqrt(n).
    Without the low half of an operand a product is off by up to 2^-12, some 1e-4."""
    c = Case(n, seed=n)
    G = np.cumsum(c.g.astype(np.float64), 0)
    memory = max(np.exp(2 * (G[t] - G[max(0, t - 400):t + 1])).sum(0).max() for t in range(0, n, 7))
    tol = 24 * 2.0 ** -24 * (1 + memory ** 0.5) + 2.0 ** -18
    with PooledAttn(CTX, 4096, max_cols=n) as pa:
        dn = c.handle(pa)
        pa.delta_write(dn, 0, 0, c.state)
        c.upload(pa)
        out, state = c.call(pa, dn, "prefill"), c.read(pa, dn)
    ref, ref_state = c.oracle()
    d = np.sqrt(((out - ref) ** 2).sum((0, 2)) / (ref ** 2).sum((0, 2)))
    s = np.sqrt(((state - ref_state) ** 2).sum((1, 2)) / (ref_state ** 2).sum((1, 2)))
    print("memory %.1f tokens: out %.2e, state %.2e of %.2e" % (memory, d.max(), s.max(), tol))
    assert tol < 2.5e-5 and d.max() <= tol and s.max() <= tol
