"""The drafted-tree calls as they are used together on the GPU: a draft written at its depths' positions, verified in one pass, its accepted path kept, and the next token behind it; the same from a
captured graph, in two contexts at once, and far behind the first 4 GB of a cache."""
import ctypes
import numpy as np
import pytest
from oracle import attn_oracle as O
from oracle import tree_oracle as T
from pooled_amd.capi import PooledAttn, PA_ERR_INVALID, tree_mask, tree_of_parents
from helpers import SHAPES
from test_gpu_graph import _hip, _ok
from test_gpu_tree import Case, random_tree
from test_tree_rules import tree_rule

pytestmark = pytest.mark.gpu
vp = ctypes.c_void_p


def depths(seen):
    return seen.sum(1) - 1


class Draft:
    """The device side of a draft's columns: pre-step inputs, positions, mask and the list of an accepted path."""

    def __init__(self, pa, d, rows, base, seen, path):
        self.base, self.n, self.m = base, seen.shape[0], len(path)
        up = lambda a: pa.to_device(np.ascontiguousarray(a))  # noqa: E731
        self.q, self.k, self.v = (up(d[x][rows]) for x in ("qraw", "kraw", "vraw"))
        self.strides = [d[x].shape[1] for x in ("qraw", "kraw", "vraw")]
        self.pos, self.mask = up((base + depths(seen)).astype(np.uint32)), up(tree_mask(seen))
        self.sel = up(np.array([len(path)] + [base + j for j in path], np.uint32))
        self.out = pa.alloc(self.n * pa.q_dim * 4)

    def write(self, pa, layer, w):
        pa.glue_kv_at(layer, self.q, self.strides[0], self.k, self.strides[1], self.v, self.strides[2], *w, self.pos, self.n, self.base, self.n)

    def verify(self, pa, layer):
        pa.attn_tree(layer, None, 0, pa.gate_buffer_ptr() if pa.cfg["gate"] else None, pa.q_dim, self.mask, (self.n + 31) // 32, self.base, self.n, self.out, pa.q_dim)

    def accept(self, pa):
        pa.kv_compact(self.base, self.sel, self.m)


def check_some(c, got, what, columns=8):
    """Some of the columns against the oracle, the first and the last among them; the others, whose sums take it too long, are numbers at least.  Besides the bound of each output, which grows
    with the context: the roundings (q, P, int8 rows' scales and products, partials, output: at most six of half a step, 2^-11) are independent, so in the norm of all outputs, which are sums of
    many terms, they add in squares: at most sqrt(6) 2^-11 < 2^-9.  A tile of 32 rows left out of 32000 would be 2^-5."""
    at = np.unique(np.concatenate([[0, c.n - 1], c.rng.integers(0, c.n, columns)]))
    ref, absolute, reach = T.tree_attention(c.q[at], c.k, c.v, c.base, c.seen[at])
    bound = T.tree_bound(ref, absolute, reach, np.abs(c.v).max(), c.base + c.n, bool(c.cfg.get("kv_q8")))
    off = np.abs(got[at] - ref)
    norm = np.sqrt((off ** 2).sum() / (ref ** 2).sum())
    print("%s base %d n %d: max-abs %.2e, %.1f %% of the bound, %.2e of the norm" % (what, c.base, c.n, off.max(), 100 * (off / bound).max(), norm), flush=True)
    assert np.isfinite(got).all() and (off <= bound).all() and norm <= 2.0 ** -9


def plain_rows(pa, layer, d, rows, base, w):
    """the rows as pa_glue_kv writes them at base, base + 1, ..."""
    q, k, v = (pa.to_device(np.ascontiguousarray(d[x][rows])) for x in ("qraw", "kraw", "vraw"))
    pa.glue_kv(layer, q, d["qraw"].shape[1], k, d["kraw"].shape[1], v, d["vraw"].shape[1], *w, base, len(rows))
    pa.sync()


def caches(pa, layer, rows):
    return [pa.kv_read(layer, t, 0, rows).tobytes() for t in range(4 if pa.cfg.get("kv_q8") else 2)]


PARENTS = [-1, 0, 0, 1, 1, 2, 3, -1, 6, 7, 8, 6, 8, 12, 13, 3, 14, 14, 5]
PATH = [0, 1, 3, 6, 8, 12, 13, 14, 17]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("base", [0, 1, 300, 2011])
def test_a_draft_is_verified_and_its_path_kept(shape, base, q8):
    """Behind the accepted path the caches of every layer have the bits, and the next token the output, that decoding the path's tokens one behind the other gives."""
    cfg = dict(SHAPES[shape], kv_q8=q8)
    seen, n, m, layers = tree_of_parents(PARENTS), len(PARENTS), len(PATH), 2
    d = O.make_inputs(cfg, 0, base + n + 1, base + 5)
    draft, next_row = list(range(base, base + n)), [base + n]
    with PooledAttn(cfg, base + n + 3, n_layers=layers, max_cols=max(base, n)) as a, PooledAttn(cfg, base + n + 3, n_layers=layers, max_cols=max(base, n)) as b:
        wa, wb = ([pa.to_device(d["qw"]), pa.to_device(d["kw"])] for pa in (a, b))
        D = Draft(a, d, draft, base, seen, PATH)
        for layer in range(layers):
            for pa, w in ((a, wa), (b, wb)):
                pa.layer_alloc(layer)
                if base:
                    plain_rows(pa, layer, d, range(base), 0, w)
            D.write(a, layer, wa)
            D.verify(a, layer)
        a.sync()
        got = D.out.download(np.float32, n * a.q_dim).reshape(n, cfg["n_heads"], cfg["head_dim"])
        parts = [a.kv_read(layers - 1, t, 0, base + n) for t in range(4 if q8 else 2)]
        kv = [O.q8_dequantize(parts[0], parts[2]), O.q8_dequantize(parts[1], parts[3])] if q8 else [p.view(np.float16).astype(np.float32) for p in parts]
        gate = a.read_gate_buffer(n) if cfg["gate"] else None
        ref, absolute, reach = T.tree_attention(a.read_q_buffer(n), *kv, base, seen, gate)
        assert (np.abs(got - ref) <= T.tree_bound(ref, absolute, reach, np.abs(kv[1]).max(), base + n, q8)).all()
        assert np.sqrt(((got - ref) ** 2).sum() / (ref ** 2).sum()) <= 2.0 ** -9               # (see check_some)
        D.accept(a)
        a.sync()
        for layer in range(layers):
            plain_rows(b, layer, d, [base + j for j in PATH], base, wb)
            assert caches(a, layer, base + m) == caches(b, layer, base + m)
        outs = []
        for pa, w in ((a, wa), (b, wb)):
            q, k, v = (pa.to_device(np.ascontiguousarray(d[x][next_row])) for x in ("qraw", "kraw", "vraw"))
            out = pa.alloc(pa.q_dim * 4)
            pa.attn_decode_step(layers - 1, q, k, v, *w, base + m, out)
            pa.sync()
            outs.append(out.download(np.float32, pa.q_dim))
        assert np.isfinite(outs[0]).all() and np.array_equal(outs[0].view(np.uint32), outs[1].view(np.uint32))


class Graph:
    def __init__(self):
        self.hip, self.stream, self.made = _hip(), vp(), []
        _ok(self.hip.hipStreamCreate(ctypes.byref(self.stream)), "hipStreamCreate")

    def record(self, calls):
        graph, gexec = vp(), vp()
        _ok(self.hip.hipStreamBeginCapture(self.stream, 0), "hipStreamBeginCapture")
        calls()
        _ok(self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph)), "hipStreamEndCapture")
        _ok(self.hip.hipGraphInstantiate(ctypes.byref(gexec), graph, None, None, 0), "hipGraphInstantiate")
        self.made.append((graph, gexec))
        return gexec

    def run(self, gexec):
        _ok(self.hip.hipGraphLaunch(gexec, self.stream), "hipGraphLaunch")
        _ok(self.hip.hipStreamSynchronize(self.stream), "hipStreamSynchronize")

    def close(self):
        for graph, gexec in self.made:
            _ok(self.hip.hipGraphExecDestroy(gexec), "hipGraphExecDestroy")
            _ok(self.hip.hipGraphDestroy(graph), "hipGraphDestroy")
        _ok(self.hip.hipStreamDestroy(self.stream), "hipStreamDestroy")


@pytest.mark.parametrize("q8", [False, True])
def test_a_draft_from_a_graph(q8):
    """Two graphs (the draft and its verification; the acceptance) replayed in turn, with eager calls between that grow the scratch both were recorded over."""
    cfg, base = dict(SHAPES["qwen36_moe"], kv_q8=q8), 3000
    seen, n = tree_of_parents(PARENTS), len(PARENTS)
    c = Case(cfg, base, n, seed=3)
    d = O.make_inputs(cfg, 0, n, 4)
    G = Graph()
    with PooledAttn(cfg, 9000, n_layers=1, max_cols=100) as pa:
        pa._chk(pa.L.pa_set_stream(pa.ctx, G.stream))
        pa.layer_alloc(0)
        context = [p[:base] for p in c.parts]
        for t, part in enumerate(context):
            pa.kv_write(0, t, 0, part)
        w = [pa.to_device(d["qw"]), pa.to_device(d["kw"])]
        D = Draft(pa, d, list(range(n)), base, seen, PATH)

        def both():
            D.write(pa, 0, w)
            D.verify(pa, 0)

        def results():
            pa.sync()
            out = D.out.download(np.float32, n * pa.q_dim).copy()
            return out, caches(pa, 0, base + n)
        both(); eager = results()
        D.accept(pa); kept = results()
        assert np.isfinite(eager[0]).all() and eager[1] != kept[1]
        draft, accept = G.record(both), G.record(lambda: D.accept(pa))
        wide_q, wide_seen = c.rng.standard_normal((100, cfg["n_heads"], cfg["head_dim"]), dtype=np.float32), random_tree(100, c.rng)
        for rep in range(4):
            D.out.upload(np.full(n * pa.q_dim, np.nan, np.float32))
            for t, part in enumerate(context):
                pa.kv_write(0, t, base, np.zeros_like(part[:n]))
            G.run(draft)
            got = results()
            assert np.array_equal(got[0].view(np.uint32), eager[0].view(np.uint32)) and got[1] == eager[1], "replay %d" % rep
            if rep > 0:                                                # an eager call with more partials than the graph's
                first = pa.run_attn_tree(0, wide_q, wide_seen, 8000, gate=wide_q)
                assert np.isfinite(first).all()
            G.run(accept)
            assert results()[1] == kept[1], "replay %d" % rep
    G.close()


@pytest.mark.parametrize("q8", [False, True])
def test_recorded_in_a_context_without_scratch(q8):
    """Nothing can be allocated under capture: the tree is not split, or into as many splits as there is room for, and a long list is walked without flags."""
    cfg, base, n = dict(SHAPES["qwen36_moe"], kv_q8=q8), 3000, 24
    c = Case(cfg, base, n, seed=6)
    rows = np.sort(c.rng.choice(base - 100, 1500, replace=False)) + 100
    G = Graph()
    for held in (0, 3):
        with c.context() as pa:
            pa._chk(pa.L.pa_set_stream(pa.ctx, G.stream))
            c.fill(pa)
            if held:                                                   # partials of three splits
                pa.set_decode_splits(held)
                pa.run_attn_tree(0, c.q, c.seen, base, gate=c.gate)
                pa.set_decode_splits(0)
            q, gate = pa.to_device(c.q.reshape(n, -1)), pa.to_device(c.gate.reshape(n, -1))
            mask, out, sel = pa.to_device(tree_mask(c.seen)), pa.alloc(n * pa.q_dim * 4), pa.to_device(np.concatenate([[rows.size], rows]).astype(np.uint32))
            tree = G.record(lambda: pa.attn_tree(0, q, pa.q_dim, gate, pa.q_dim, mask, 1, base, n, out, pa.q_dim))
            cut = G.record(lambda: pa.kv_compact(100, sel, 2000))
            for rep in range(3):
                out.upload(np.full(n * pa.q_dim, np.nan, np.float32))
                for t, part in enumerate(c.parts):
                    pa.kv_write(0, t, 0, part)
                G.run(tree)
                c.check(out.download(np.float32, n * pa.q_dim).reshape(c.q.shape), what="recorded with %d splits' scratch" % held)
                G.run(cut)
                for t, part in enumerate(c.parts):
                    got = pa.kv_read(0, t, 0, base + n)
                    assert got.tobytes() == T.compact(part, 100, rows).tobytes(), (rep, t)
    G.close()


def test_two_contexts_on_two_streams():
    """Calls of two contexts enqueued in turn without a wait between them: each gives what it gives alone."""
    cases = [Case(SHAPES["qwen36_moe"], 5000, 24, seed=1), Case(dict(SHAPES["qwen3_1p7b"], kv_q8=True), 3000, 40, seed=2)]
    graphs = [Graph(), Graph()]
    with cases[0].context() as a, cases[1].context() as b:
        work = []
        for pa, c, g in ((a, cases[0], graphs[0]), (b, cases[1], graphs[1])):
            pa._chk(pa.L.pa_set_stream(pa.ctx, g.stream))
            c.fill(pa)
            alone = pa.run_attn_tree(0, c.q, c.seen, c.base, gate=c.gate)
            gate = pa.to_device(c.gate.reshape(c.n, -1)) if c.gate is not None else None
            outs = [pa.alloc(c.n * pa.q_dim * 4) for _ in range(6)]
            work.append((pa, c, alone, pa.to_device(c.q.reshape(c.n, -1)), gate, pa.to_device(tree_mask(c.seen)), outs))
        for i in range(6):
            for pa, c, _, q, gate, mask, outs in work:
                pa.attn_tree(0, q, pa.q_dim, gate, pa.q_dim, mask, (c.n + 31) // 32, c.base, c.n, outs[i], pa.q_dim)
        for pa, c, alone, _, _, _, outs in work:
            pa.sync()
            for o in outs:
                assert np.array_equal(o.download(np.uint32, alone.size), alone.view(np.uint32).ravel())
    for g in graphs:
        g.close()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 128), (6, 1, 256), (20, 1, 128), (3, 3, 256)])
@pytest.mark.parametrize("n,base,splits", [(150, 40, 1), (333, 3, 1), (333, 300, 0), (700, 65, 2), (1001, 30, 0)])
def test_drafts_wider_than_the_windows_of_masks(heads, kv_heads, hd, n, base, splits, q8):
    """More drafted rows than a workgroup keeps mask words of at a time, seen through random patterns."""
    cfg = dict(n_heads=heads, n_kv_heads=kv_heads, head_dim=hd, n_rot=64, rope_theta=1e6, eps=1e-6, qk_norm=True, gate=False, kv_q8=q8)
    c = Case(cfg, base, n, seed=n + heads)
    c.seen = c.rng.random((n, n)) < 0.02
    c.seen[np.arange(n), np.arange(n)] = True
    with c.context() as pa:
        c.fill(pa)
        pa.set_decode_splits(splits)
        check_some(c, pa.run_attn_tree(0, c.q, c.seen, base), "%d / %d of %d" % (heads, kv_heads, hd), 40)


def test_other_columns_masks_do_not_matter():
    """A column's output keeps within rounding of itself, whatever the others see (a column that sees nothing but zeros aside, both are checked against the oracle)."""
    c = Case(SHAPES["qwen36_moe"], 500, 30, seed=9)
    with c.context() as pa:
        c.fill(pa)
        first = pa.run_attn_tree(0, c.q, c.seen, c.base, gate=c.gate)
        other = c.seen.copy()
        other[::2] = c.rng.random((15, 30)) < 0.5
        second = pa.run_attn_tree(0, c.q, other, c.base, gate=c.gate)
        c.check(first)
        c.check(second, seen=other)
        ref, absolute, reach = T.tree_attention(c.q, c.k, c.v, c.base, c.seen, c.gate)
        assert (np.abs(first - second)[1::2] <= 2 * T.tree_bound(ref, absolute, reach, np.abs(c.v).max(), 530)[1::2]).all()


def test_a_key_that_is_not_a_number():
    """A drafted key row with NaN makes the columns that see it NaN, whoever else shares their block, and no other."""
    for base, n, splits in ((40, 20, 0), (2000, 20, 0), (0, 33, 1)):
        c = Case(SHAPES["qwen3_1p7b"], base, n, seed=base)
        at = n // 2
        parts = [p.copy() for p in c.parts]
        parts[0][base + at] = 0x7E00
        with c.context() as pa:
            c.fill(pa)
            pa.set_decode_splits(splits)
            clean = pa.run_attn_tree(0, c.q, c.seen, base)
            pa.kv_write(0, 0, 0, parts[0])
            got = pa.run_attn_tree(0, c.q, c.seen, base)
        sees = c.seen[:, at]
        assert sees.any() and not sees.all()
        assert np.isnan(got[sees]).all()
        ref, absolute, reach = T.tree_attention(c.q, c.k, c.v, base, c.seen)
        assert (np.abs(got - ref) <= T.tree_bound(ref, absolute, reach, np.abs(c.v).max(), base + n))[~sees].all() and np.isfinite(clean).all()


def test_axes_may_change_between_calls():
    """pa_set_rope_axes holds from call to call; a graph keeps the axes that it was recorded with."""
    cfg, n = SHAPES["qwen36_moe"], 6
    half = cfg["n_rot"] // 2
    d = O.make_inputs(cfg, 0, n, 1)
    pos = np.random.default_rng(2).integers(0, 500, (4, n)).astype(np.uint32)
    G = Graph()
    with PooledAttn(cfg, 600, n_layers=1, max_cols=n) as pa:
        pa._chk(pa.L.pa_set_stream(pa.ctx, G.stream))
        pa.layer_alloc(0)
        w = [pa.to_device(d["qw"]), pa.to_device(d["kw"])]
        q, k, v = (pa.to_device(d[x]) for x in ("qraw", "kraw", "vraw"))
        p = pa.to_device(pos)

        def call():
            pa.glue_kv_at(0, q, d["qraw"].shape[1], k, d["kraw"].shape[1], v, d["vraw"].shape[1], *w, p, n, 0, n)

        def reads(axis):
            ref = T.glue_at(d["qraw"], d["kraw"], d["vraw"], d["qw"], d["kw"], pos[:axis.max() + 1], axis, cfg)
            pa.sync()
            return np.array_equal(pa.read_q_buffer(n).view(np.uint32), ref["q"].view(np.uint32))
        one, three = np.zeros(half, int), np.arange(half) % 3
        call(); assert reads(one)
        pa.set_rope_axes(three)
        recorded = G.record(call)
        pa.set_rope_axes(np.arange(half) % 4); call(); assert reads(np.arange(half) % 4)
        for _ in range(3):
            pa.set_rope_axes(None); call(); assert reads(one)
            G.run(recorded); assert reads(three)
    G.close()


def test_rows_behind_the_first_4_gb_of_a_cache():
    """One key head of 256 over 8.4 million rows of f16: rows behind 2^32 bytes are written, seen and moved.  Nearly all rows are zeros, so the sums are those of a few rows."""
    base, n, hd, heads = (1 << 23) + 70000, 9, 256, 4
    assert base * hd * 2 > 1 << 32
    cfg = dict(n_heads=heads, n_kv_heads=1, head_dim=hd, n_rot=32, rope_theta=1e6, eps=1e-6, qk_norm=False, gate=False)
    rng = np.random.default_rng(12)
    seen = random_tree(n, rng, 0.4)
    with PooledAttn(cfg, base + n + 5, n_layers=1, max_cols=n) as pa:
        pa.layer_alloc(0)
        at = np.sort(np.array([3, 4000000, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 23) + 60000, base - 1]))
        # the columns' q all point the same way, nearly, and the rows too: scores of 14, against 8.4 million of 0
        way = rng.standard_normal(hd); way /= np.sqrt((way ** 2).sum())
        q = (15 * way + 0.05 * rng.standard_normal((n, heads, hd))).astype(np.float32)
        k = O.f16_round((15 * way + 0.05 * rng.standard_normal((at.size, 1, hd))).astype(np.float32))
        v = O.f16_round(rng.standard_normal((at.size, 1, hd), dtype=np.float32))
        for i, row in enumerate(at):
            pa.kv_write(0, 0, int(row), O.f16_bits(k[i:i + 1])); pa.kv_write(0, 1, int(row), O.f16_bits(v[i:i + 1]))
        # the draft, at positions 0, which turn nothing
        dk, dv = (15 * way + 0.05 * rng.standard_normal((n, hd))).astype(np.float32), rng.standard_normal((n, hd), dtype=np.float32)
        pos = np.zeros((1, n), np.uint32)
        ins = [pa.to_device(x) for x in (q.reshape(n, -1), dk, dv)]
        pa.glue_kv_at(0, ins[0], heads * hd, ins[1], hd, ins[2], hd, None, None, pa.to_device(pos), n, base, n)
        pa.sync()
        K = np.concatenate([k, O.f16_round(dk).reshape(n, 1, hd)]); V = np.concatenate([v, O.f16_round(dv).reshape(n, 1, hd)])
        assert np.array_equal(pa.kv_read(0, 0, base, n), O.f16_bits(K[at.size:])) and np.array_equal(pa.kv_read(0, 1, base, n), O.f16_bits(V[at.size:]))
        splits = 256
        pa.set_decode_splits(splits)
        got = pa.run_attn_tree(0, q, seen, base)
        zeros = base - at.size
        ref, absolute, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, heads))
        for c in range(n):
            t = np.concatenate([np.ones(at.size, bool), seen[c]])
            for h in range(heads):
                s = K[t, 0].astype(np.float64) @ q[c, h] / 16
                w = np.exp(s)
                ref[c, h], absolute[c, h] = (w @ V[t, 0]) / (w.sum() + zeros), (w @ np.abs(V[t, 0].astype(np.float64))) / (w.sum() + zeros)
                reach[c, h] = (np.abs(K[t, 0].astype(np.float64)) @ np.abs(q[c, h])).max() / 16
        # (small weights are rounded against their own split's largest: the rows of a split count, not those of the cache; and the zero rows' weights, of which `absolute` holds nothing, move the
        # denominator by as much as they move themselves: exactly 1 each in a split of zeros, off by 2^-25 of that split's largest elsewhere, which the same term covers)
        bound = T.tree_bound(ref, absolute, reach, np.abs(V).max(), -(-(base + n) // splits) + 32)
        off = np.abs(got - ref)
        print("far rows: max-abs %.2e of %.2e, outputs up to %.2f, %.1f %% of the bound" % (off.max(), bound.min(), np.abs(ref).max(), 100 * (off / bound).max()))
        assert (off <= bound).all() and np.abs(ref).max() > 5 * bound.max()
        keep = [1 << 23, (1 << 23) + 1, (1 << 23) + 60000, base - 1, base + 2, base + 8]
        pa.run_kv_compact((1 << 23) - 1, keep)
        where = [3, 4, 5, 6, at.size + 2, at.size + 8]
        for t, whole in ((0, K), (1, V)):
            assert np.array_equal(pa.kv_read(0, t, (1 << 23) - 1, 6), O.f16_bits(whole[where]))
            assert np.array_equal(pa.kv_read(0, t, base, n), O.f16_bits(whole[at.size:]))


@pytest.mark.parametrize("heads,kv_heads,hd,n,base,splits,q8", [
    (64, 8, 128, 17, 16000, 0, False), (16, 8, 128, 65, 16000, 0, False), (16, 2, 128, 33, 32000, 0, False), (64, 1, 128, 130, 500, 4, False),
    (16, 2, 128, 17, 32000, 0, True), (16, 8, 128, 65, 8000, 0, True), (16, 2, 128, 33, 16000, 0, True), (64, 8, 128, 130, 100, 4, True),
    (16, 8, 256, 100, 32000, 0, False), (64, 8, 256, 33, 8000, 0, False), (64, 8, 256, 130, 500, 4, False)])
def test_two_blocks_of_rows_a_wave(heads, kv_heads, hd, n, base, splits, q8):
    """The plans whose waves hold 32 stacked rows: one group and several, drafts within a window of masks and wider."""
    cfg = dict(n_heads=heads, n_kv_heads=kv_heads, head_dim=hd, n_rot=64, rope_theta=1e6, eps=1e-6, qk_norm=True, gate=False, kv_q8=q8)
    assert tree_rule(cfg, base, n, splits)[0] == 2
    c = Case(cfg, base, n, seed=n)
    with c.context() as pa:
        c.fill(pa)
        pa.set_decode_splits(splits)
        check_some(c, pa.run_attn_tree(0, c.q, c.seen, base), "%d / %d of %d" % (heads, kv_heads, hd))


@pytest.mark.parametrize("heads,hd,q8", [(64, 128, False), (64, 128, True), (32, 256, False)])
def test_two_blocks_of_rows_a_wave_without_splits(heads, hd, q8):
    cfg = dict(n_heads=heads, n_kv_heads=1, head_dim=hd, n_rot=64, rope_theta=1e6, eps=1e-6, qk_norm=True, gate=False, kv_q8=q8)
    n, base = 1000 if hd == 128 else 1500, 0
    plan = tree_rule(cfg, base, n)
    assert plan[0] == 2 and plan[4] == 1
    c = Case(cfg, base, n, seed=hd)
    with c.context() as pa:
        c.fill(pa)
        check_some(c, pa.run_attn_tree(0, c.q, c.seen, base), "%d / 1 of %d, one split" % (heads, hd))


@pytest.mark.parametrize("q8", [False, True])
def test_long_lists_one_behind_the_other_and_from_a_graph(q8):
    """Lists of segments that wait for one another: several lengths and limits in turn, eagerly and replayed, each as if it were the first call."""
    cfg, seq = dict(SHAPES["qwen36_moe"], kv_q8=q8), 6000
    c = Case(cfg, seq - 1, 1, seed=8, more=0)
    G = Graph()
    with PooledAttn(cfg, seq, n_layers=1, max_cols=1) as pa:
        pa._chk(pa.L.pa_set_stream(pa.ctx, G.stream))
        pa.layer_alloc(0)
        calls = []
        for dst, n, limit in ((0, 3000, 6000), (7, 300, 400), (100, 2900, 2900), (3, 0, 5000), (1, 5000, 5999), (0, 257, 257)):
            rows = np.sort(c.rng.choice(seq - dst, n, replace=False)) + dst
            calls.append((dst, rows, limit, pa.to_device(np.concatenate([[n], rows]).astype(np.uint32))))

        def once(run, dst, rows):
            for t, part in enumerate(c.parts):
                pa.kv_write(0, t, 0, part)
            run()
            pa.sync()
            for t, part in enumerate(c.parts):
                assert pa.kv_read(0, t, 0, seq).tobytes() == T.compact(part, dst, rows).tobytes(), (dst, len(rows), t)
        for dst, rows, limit, sel in calls + calls[::-1]:
            once(lambda: pa.kv_compact(dst, sel, limit), dst, rows)
        recorded = [(G.record(lambda: pa.kv_compact(dst, sel, limit)), dst, rows) for dst, rows, limit, sel in calls]
        for rep in range(3):
            for graph, dst, rows in recorded:
                once(lambda: G.run(graph), dst, rows)
            dst, rows, limit, sel = calls[rep]
            once(lambda: pa.kv_compact(dst, sel, limit), dst, rows)
    G.close()


def test_inputs_in_the_buffers_that_the_pre_step_writes():
    cfg, n = SHAPES["qwen36_moe"], 4
    d = O.make_inputs(cfg, 0, n, 1)
    with PooledAttn(cfg, 64, n_layers=1, max_cols=n) as pa:
        pa.layer_alloc(0)
        w, (q, k, v) = [pa.to_device(d["qw"]), pa.to_device(d["kw"])], (pa.to_device(d[x]) for x in ("qraw", "kraw", "vraw"))
        p = pa.to_device(np.arange(n, dtype=np.uint32))
        for buf in (pa.q_buffer_ptr(), pa.gate_buffer_ptr()):
            for at in range(4):
                ptrs = [q.ptr, k.ptr, v.ptr, p.ptr]
                ptrs[at] = buf + 64
                rc = pa.L.pa_glue_kv_at(pa.ctx, 0, ptrs[0], d["qraw"].shape[1], ptrs[1], d["kraw"].shape[1], ptrs[2], d["vraw"].shape[1], w[0].ptr, w[1].ptr, ptrs[3], n, 0, n)
                assert rc == PA_ERR_INVALID


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd,n_rot", [(5, 5, 128, 128), (6, 3, 128, 64), (7, 1, 128, 96), (3, 1, 256, 64), (9, 3, 256, 256), (1, 1, 256, 16)])
def test_the_pre_step_of_head_counts_that_fill_no_wave(heads, kv_heads, hd, n_rot, gate, q8):
    """A wave takes 512 values of heads: the last one of a column may have fewer.  The bits of pa_glue_kv, and nothing beside them written."""
    cfg = dict(n_heads=heads, n_kv_heads=kv_heads, head_dim=hd, n_rot=n_rot, rope_theta=1e6, eps=1e-6, qk_norm=True, gate=gate, kv_q8=q8)
    base, n = 11, 13
    d = O.make_inputs(cfg, 0, n, heads)
    got = []
    for at in (False, True):
        with PooledAttn(cfg, base + n + 3, n_layers=1, max_cols=n + 2) as pa:
            pa.layer_alloc(0)
            w, (q, k, v) = [pa.to_device(d["qw"]), pa.to_device(d["kw"])], [pa.to_device(d[x]) for x in ("qraw", "kraw", "vraw")]
            fill = np.full((n + 2) * pa.q_dim, 7.0, np.float32)
            for buf in (pa.q_buffer_ptr(), pa.gate_buffer_ptr() if gate else None):
                if buf:
                    pa._chk(pa.L.pa_upload(pa.ctx, buf, fill.ctypes.data, fill.nbytes))
            if at:
                pa.glue_kv_at(0, q, d["qraw"].shape[1], k, d["kraw"].shape[1], v, d["vraw"].shape[1], *w, pa.to_device((base + np.arange(n)).astype(np.uint32)), n, base, n)
            else:
                pa.glue_kv(0, q, d["qraw"].shape[1], k, d["kraw"].shape[1], v, d["vraw"].shape[1], *w, base, n)
            pa.sync()
            got.append([pa.read_q_buffer(n + 2).tobytes(), pa.read_gate_buffer(n + 2).tobytes() if gate else b""] + caches(pa, 0, base + n + 3))
    assert got[0] == got[1]


def test_two_contexts_cut_long_caches_at_once():
    """Compactions of more segments than the device runs at a time, of two contexts on two streams, enqueued in turn without a wait between them."""
    seq, graphs, work = 150000, [Graph(), Graph()], []
    rng = np.random.default_rng(4)
    cfgs = [dict(n_heads=h, n_kv_heads=h, head_dim=128, n_rot=128, rope_theta=1e6, eps=1e-6, qk_norm=False, gate=False) for h in (1, 3)]
    with PooledAttn(cfgs[0], seq, n_layers=1, max_cols=1) as a, PooledAttn(cfgs[1], seq, n_layers=1, max_cols=1) as b:
        for pa, g in ((a, graphs[0]), (b, graphs[1])):
            pa._chk(pa.L.pa_set_stream(pa.ctx, g.stream))
            pa.layer_alloc(0)
            parts = [rng.integers(0, 1 << 16, (seq, pa.cfg["n_kv_heads"], 128), dtype=np.uint16) for _ in range(2)]
            for t in range(2):
                pa.kv_write(0, t, 0, parts[t])
            lists = [np.sort(rng.choice(n - 5, m, replace=False)) + 5 for n, m in ((seq, 120000), (120000, 100000), (100000, 90000))]
            work.append((pa, parts, lists, [pa.to_device(np.concatenate([[x.size], x]).astype(np.uint32)) for x in lists]))
        for i in range(3):
            for pa, _, lists, sels in work:
                pa.kv_compact(5, sels[i], lists[i].size)
        for pa, parts, lists, _ in work:
            pa.sync()
            for t in range(2):
                want = parts[t]
                for rows in lists:
                    want = T.compact(want, 5, rows)
                assert pa.kv_read(0, t, 0, seq).tobytes() == want.tobytes()
    for g in graphs:
        g.close()
