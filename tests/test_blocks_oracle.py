"""The 64-bit oracle of the blocks beside attention against answers that are known without it."""
import numpy as np
from oracle import attn_oracle as A
from oracle import blocks_oracle as B


def test_delta_rule_one_token_by_hand():
    S = np.array([[[1., 2.], [3., 4.]]])                               # [1 head, 2 values, 2 keys]
    out, S1 = B.delta_rule(np.array([[[1., 1.]]]), np.array([[[0.5, 0.]]]), np.array([[[1., 1.]]]), np.log([[0.5]]), np.array([[2.]]), S, scale=1., l2norm=False)
    # S' = S / 2; u = 2 (1 - S' k) = 2 (1 - 0.25), 2 (1 - 0.75)
    want = np.array([[0.5 + 1.5 * 0.5, 1.], [1.5 + 0.5 * 0.5, 2.]])
    assert np.allclose(S1[0], want) and np.allclose(out[0, 0], want.sum(1))


def test_delta_rule_stores_values_under_orthogonal_keys():
    rng = np.random.default_rng(0)
    v = rng.standard_normal((4, 1, 3))
    keys = np.eye(4)[:, None, :]
    out, S = B.delta_rule(keys, keys, v, np.zeros((4, 1)), np.ones((4, 1)), np.zeros((1, 3, 4)), scale=1., eps=0.)
    assert np.allclose(S[0].T, v[:, 0]) and np.allclose(out, v)
    again, S2 = B.delta_rule(keys[1:2], keys[1:2], v[:1], np.zeros((1, 1)), np.ones((1, 1)), S, scale=1., eps=0.)      # overwriting key 1
    assert np.allclose(S2[0, :, 1], v[0, 0]) and np.allclose(S2[0, :, 0], v[0, 0]) and np.allclose(S2[0, :, 2], v[2, 0])


def test_delta_rule_left_out_and_emptied():
    rng = np.random.default_rng(1)
    n, nk, nv, hk, hv = 5, 1, 2, 4, 3
    q, k, v = rng.standard_normal((n, nk, hk)), rng.standard_normal((n, nk, hk)), rng.standard_normal((n, nv, hv))
    g, beta, S = -rng.random((n, nv)), rng.random((n, nv)), rng.standard_normal((nv, hv, hk))
    beta[2] = 0; g[2] = 0
    keep = [0, 1, 3, 4]
    assert np.allclose(B.delta_rule(q, k, v, g, beta, S)[1], B.delta_rule(q[keep], k[keep], v[keep], g[keep], beta[keep], S)[1])
    g[3] = -np.inf
    assert np.allclose(B.delta_rule(q, k, v, g, beta, S)[1], B.delta_rule(q[3:], k[3:], v[3:], g[3:], beta[3:], np.zeros_like(S))[1])
    assert np.allclose(B.delta_rule(q, k, v, g, beta, S, commit=2)[1], B.delta_rule(q[:2], k[:2], v[:2], g[:2], beta[:2], S)[1])


def test_delta_rule_equals_the_chunked_solution():
    rng = np.random.default_rng(2)
    n, hk, hv = 16, 8, 5
    q, k, v = rng.standard_normal((n, 1, hk)), rng.standard_normal((n, 1, hk)), rng.standard_normal((n, 1, hv))
    g, beta, S = -0.3 * rng.random((n, 1)), rng.random((n, 1)), rng.standard_normal((1, hv, hk))
    out, S1 = B.delta_rule(q, k, v, g, beta, S)
    unit = lambda a: a[:, 0] / np.sqrt((a[:, 0] ** 2).sum(-1, keepdims=True) + 1e-6)  # noqa: E731
    Q, K, V, G, b = unit(q) * hk ** -0.5, unit(k), v[:, 0], np.cumsum(g[:, 0]), beta[:, 0]
    D = np.exp(np.tril(G[:, None] - G[None]))
    T = np.linalg.inv(np.eye(n) + np.tril(b[:, None] * D * (K @ K.T), -1))
    X = b[:, None] * (V - np.exp(G)[:, None] * (K @ S[0].T))
    assert np.allclose(out[:, 0], np.exp(G)[:, None] * (Q @ S[0].T) + np.tril(D * (Q @ K.T)) @ T @ X)
    assert np.allclose(S1[0].T, np.exp(G[-1]) * S[0].T + (np.exp(G[-1] - G)[:, None] * K).T @ T @ X)


def test_delta_glue_known_points():
    rng = np.random.default_rng(3)
    n, ch, nv = 7, 8, 2
    x, a, b = rng.standard_normal((n, ch)), rng.standard_normal((n, nv)), rng.standard_normal((n, nv))
    w1 = rng.standard_normal((ch, 1))
    y, g, beta, st = B.delta_glue(x, w1, None, np.zeros((n, nv)), np.zeros((n, nv)), np.zeros(nv), np.zeros(nv), np.zeros((0, ch)))
    z = x * w1[:, 0]
    assert np.allclose(y, z / (1 + np.exp(-z))) and np.allclose(g, -np.log(2)) and np.allclose(beta, 0.5) and st.shape == (0, ch)
    w, s0 = rng.standard_normal((ch, 4)), rng.standard_normal((3, ch))
    whole = B.delta_glue(x, w, None, a, b, np.zeros(nv), np.zeros(nv), s0)
    for cut in (1, 2, 5):
        first = B.delta_glue(x[:cut], w, None, a[:cut], b[:cut], np.zeros(nv), np.zeros(nv), s0)
        rest = B.delta_glue(x[cut:], w, None, a[cut:], b[cut:], np.zeros(nv), np.zeros(nv), first[3])
        assert np.allclose(np.concatenate([first[0], rest[0]]), whole[0]) and np.allclose(rest[3], whole[3])
        assert np.allclose(B.delta_glue(x, w, None, a, b, np.zeros(nv), np.zeros(nv), s0, commit=cut)[3], first[3])


def _experts(rng, E, dim, ffn):
    return dict(gate=rng.standard_normal((E, ffn, dim)), up=rng.standard_normal((E, ffn, dim)), down=rng.standard_normal((E, dim, ffn)))


def test_moe_layer_dense_single_and_ties():
    rng = np.random.default_rng(4)
    E, dim, ffn, n = 4, 32, 32, 3
    ex = {k: a.astype(np.float32) for k, a in _experts(rng, E, dim, ffn).items()}
    x, router = rng.standard_normal((n, dim)), rng.standard_normal((E, dim)).astype(np.float32)
    silu = lambda z: z / (1 + np.exp(-z))  # noqa: E731
    ffnet = lambda e, v: ex["down"][e] @ (silu(ex["gate"][e] @ v) * (ex["up"][e] @ v))  # noqa: E731
    y, ids, w = B.moe_layer(x, None, router, ex, E, A.W_F32, norm_topk=False)
    for t in range(n):
        p = np.exp(router @ x[t]); p /= p.sum()
        assert np.allclose(y[t], x[t] + sum(p[e] * ffnet(e, x[t]) for e in range(E)))
        assert np.allclose(w[t], np.sort(p)[::-1])
    y, ids, w = B.moe_layer(x, None, router, ex, 1, A.W_F32, norm_topk=True)
    assert np.allclose(w, 1) and np.allclose(y[0], x[0] + ffnet(ids[0, 0], x[0]))
    same = np.repeat(router[:1], E, 0)
    assert B.moe_layer(x, None, same, ex, 2, A.W_F32)[1].tolist() == [[0, 1]] * n
