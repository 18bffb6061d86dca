"""CPU oracle of the drafted-tree calls (numpy, 64 bits): attention of a tree over a cache, the pre-step with positions of each column's own, compaction.
TEST INFRASTRUCTURE ONLY; written from the formulas in include/pooled_attn.h.

How each function is pinned (tests/test_tree_rules.py):
  tree_attention   a triangular mask equals attn_oracle.attention; two rows by hand; a column that sees nothing gives zeros
  glue_at          one axis that holds base + c equals attn_oracle.glue_kv; axes that agree equal one axis; a pair turns by its own axis alone
  compact          against a loop over the list that copies row by row
"""
import numpy as np
from oracle import attn_oracle as O


def tree_attention(q, k, v, base, seen, gate=None):
    """q [n, nH, hd]; seen bool [n, m] of m drafted rows (n of their columns, or all); k, v numbers [>= base + m, nKV, hd] -> (out [n, nH, hd] f64, absolute [n, nH, hd]: sum p |v|, reach [n, nH]: the largest sum |q_i k_i| / sqrt(hd) of a seen row)."""
    q = np.asarray(q, np.float64)
    n, nH, hd = q.shape
    T, nKV = base + np.shape(seen)[1], k.shape[1]
    k, v = np.asarray(k[:T], np.float64), np.asarray(v[:T], np.float64)
    full = np.concatenate([np.ones((n, base), bool), np.asarray(seen, bool)], 1)
    out, absolute, reach = np.zeros((n, nH, hd)), np.zeros((n, nH, hd)), np.zeros((n, nH))
    for h in range(nH):
        kh, vh = k[:, h // (nH // nKV)], v[:, h // (nH // nKV)]
        for c in range(n):
            t = np.nonzero(full[c])[0]
            if t.size == 0:
                continue
            s = kh[t] @ q[c, h] / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[c, h], absolute[c, h] = p @ vh[t], p @ np.abs(vh[t])
            reach[c, h] = (np.abs(kh[t]) @ np.abs(q[c, h])).max() / np.sqrt(hd)
    if gate is not None:
        g = 1 / (1 + np.exp(-np.asarray(gate, np.float64)))
        out, absolute = out * g, absolute * g
    return out, absolute, reach


def tree_bound(out, absolute, reach, v_max, rows, q8=False, out_f16=False):
    """How far pa_attn_tree may be from tree_attention, by the roundings that it makes (f16: half a step is 2^-11 of the value, or 2^-25 of what is below 2^-14):
      q is rounded to f16, and so are int8 rows' values (2^-11 of themselves, and 2^-20 for the parts of the scale: kv, 2^-10, is more than both; those below 2^-14 by up to 2^-24 each,
      which is not in here), and a product of hd terms is summed in f32: a score is off by at most
        ds = reach (2^-11 + kv + 2^-16)  -- hd 2^-24 <= 2^-16 for the sums
      a weight is off by e^ds and by the rounding of P, numerator and denominator each; exp2 and the f32 sums add less than 2^-16; P below 2^-14 are off by 2^-25 each, of a sum of
        about 1 at the least (a row's reference is one of its own scores, whose weight is in the sum)
      value rows of int8 caches are off by kv; the output is rounded if it is f16, and so may the partials of splits be."""
    half, kv = 2.0 ** -11, 2.0 ** -10 if q8 else 0.0
    ds = reach[..., None] * (half + kv + 2.0 ** -16)
    w = np.exp(2 * ds) * (1 + half) ** 2 * (1 + 2.0 ** -16) - 1
    tiny = (rows + 2) * 2.0 ** -25 * v_max
    return absolute * (1 + w) * (1 + kv) * (1 + half) * (1 + (half if out_f16 else 0)) - absolute + 2 * tiny + 2.0 ** -24


def glue_at(q_in, k_in, v_in, qw, kw, pos, axis, cfg):
    """The pre-step at positions pos [axes, n]; axis [n_rot / 2].  Returns dict(q f32 [n, nH, hd], gate or None, k, v f32 [n, nKV, hd]), the arithmetic of attn_oracle.glue_kv."""
    n, nH, nKV, hd, half = q_in.shape[0], cfg["n_heads"], cfg["n_kv_heads"], cfg["head_dim"], cfg["n_rot"] // 2
    q, gate = O.qsplit(q_in, nH, hd) if cfg.get("gate") else (np.asarray(q_in, np.float32).reshape(n, nH, hd), None)
    k = np.asarray(k_in, np.float32).reshape(n, nKV, hd)
    if cfg.get("qk_norm", True):
        q, k = O.head_rmsnorm(q, qw, cfg["eps"]), O.head_rmsnorm(k, kw, cfg["eps"])
    at = np.asarray(pos)[np.asarray(axis)].T.astype(np.float32)                       # [n, half]
    angle = (at * O.rope_inv_freq(cfg["n_rot"], cfg["rope_theta"])).astype(np.float32).astype(np.float64)
    c, s = np.cos(angle).astype(np.float32)[:, None], np.sin(angle).astype(np.float32)[:, None]

    def turn(x):
        y = np.array(x, np.float32)
        a, b = y[..., :half].copy(), y[..., half:2 * half].copy()
        y[..., :half] = (a * c).astype(np.float32) - (b * s).astype(np.float32)
        y[..., half:2 * half] = (b * c).astype(np.float32) + (a * s).astype(np.float32)
        return y
    return dict(q=turn(q), gate=gate, k=turn(k), v=np.asarray(v_in, np.float32).reshape(n, nKV, hd))


def compact(cache, dst, rows):
    """cache [rows, ...] with row dst + i taken from row rows[i], all read before any is written."""
    out = np.array(cache)
    out[dst:dst + len(rows)] = np.asarray(cache)[np.asarray(rows, np.int64)] if len(rows) else out[dst:dst]
    return out
