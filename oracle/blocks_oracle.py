"""CPU oracle of the blocks beside attention (numpy, 64 bits): the gated delta rule, its pre-step, the mixture of experts.
TEST INFRASTRUCTURE ONLY; written from the formulas in include/pooled_attn.h.

How each function is pinned (tests/test_blocks_oracle.py):
  delta_rule   one token by hand; no decay and unit steps over orthogonal keys store values exactly; beta 0 leaves a token out;
               g = -inf empties the state; the chunked solution of the triangular system gives the same numbers
  delta_glue   a width-1 filter is a product; a call in two halves equals one call; softplus and sigmoid at known points
  moe_layer    top_k = n_experts without renormalisation equals the dense mixture; one expert is a plain feed-forward; ties go to the
               lowest index
"""
import numpy as np
from oracle import attn_oracle as O


def sigmoid(x):
    x = np.asarray(x, np.float64)
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1 / (1 + e), e / (1 + e))


def delta_rule(q, k, v, g, beta, state, scale=None, l2norm=True, eps=1e-6, commit=None):
    """q, k [n, nk, hk], v [n, nv, hv], g, beta [n, nv], state [nv, hv, hk] -> out [n, nv, hv], state after `commit` (default all) columns."""
    q, k, v, g, beta = (np.asarray(a, np.float64) for a in (q, k, v, g, beta))
    S = np.array(state, np.float64)
    n, nk, hk = k.shape
    nv = v.shape[1]
    commit = n if commit is None else commit
    if l2norm:
        q = q / np.sqrt((q ** 2).sum(-1, keepdims=True) + eps)
        k = k / np.sqrt((k ** 2).sum(-1, keepdims=True) + eps)
    q = q * (hk ** -0.5 if not scale else scale)
    of = np.arange(nv) // (nv // nk)
    out, kept = np.empty((n, nv, v.shape[2])), S.copy()
    for t in range(n):
        kt, qt = k[t][of], q[t][of]
        S = np.exp(g[t])[:, None, None] * S
        u = beta[t][:, None] * (v[t] - np.einsum("hvk,hk->hv", S, kt))
        S = S + u[:, :, None] * kt[:, None, :]
        out[t] = np.einsum("hvk,hk->hv", S, qt)
        if t + 1 == commit:
            kept = S.copy()
    return out, kept


def delta_glue(qkv, w, bias, a, b, a_log, dt_bias, state, commit=None):
    """qkv [n, ch], w [ch, W], state [W - 1, ch] -> silu(conv) [n, ch], g [n, nv], beta [n, nv], new state."""
    x = np.concatenate([np.asarray(state, np.float64).reshape(-1, qkv.shape[1]), np.asarray(qkv, np.float64)])
    n, W = qkv.shape[0], w.shape[1]
    commit = n if commit is None else commit
    y = np.zeros((n, qkv.shape[1])) + (0 if bias is None else np.asarray(bias, np.float64))
    for j in range(W):
        y = y + x[j:j + n] * np.asarray(w, np.float64)[:, j]
    z = np.asarray(a, np.float64) + np.asarray(dt_bias, np.float64)
    g = -np.exp(np.asarray(a_log, np.float64)) * np.logaddexp(0, z)
    return y * sigmoid(y), g, sigmoid(b), x[commit:commit + W - 1]


def moe_layer(x, norm_w, router, experts, top_k, kind, norm_topk=True, shared=None, eps=1e-6):
    """x [n, dim] -> y [n, dim], ids [n, top_k], weights [n, top_k].  experts / shared: the dicts of PooledAttn.moe."""
    x = np.asarray(x, np.float64)
    n, E = x.shape[0], router.shape[0]
    xn = x if norm_w is None else x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.asarray(norm_w, np.float64)
    logits = xn @ np.asarray(router, np.float64).T
    p = np.exp(logits - logits.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    ids = np.argsort(-logits, axis=-1, kind="stable")[:, :top_k]         # not of p: distinct logits have distinct probabilities, also where exp underflows
    w = np.take_along_axis(p, ids, 1)
    if norm_topk:
        w = w / w.sum(-1, keepdims=True)

    def wide(d, name, e=None):
        pick = (lambda a: a) if e is None else (lambda a: a[e])
        return O.w_dequant(kind, pick(d[name]), None if kind == O.W_F32 else pick(d[name + "_s"])).astype(np.float64)

    def expert(v, gate, up, down):
        a = gate @ v
        return down @ (a * sigmoid(a) * (up @ v))
    y = x.copy()
    for e in np.unique(ids):
        mats = [wide(experts, m, e) for m in ("gate", "up", "down")]
        for t, r in zip(*np.nonzero(ids == e)):
            y[t] += w[t, r] * expert(xn[t], *mats)
    if shared is not None:
        mats = [wide(shared, m) for m in ("gate", "up", "down")]
        for t in range(n):
            y[t] += sigmoid(xn[t] @ np.asarray(shared["weight"], np.float64)) * expert(xn[t], *mats)
    return y, ids, w
