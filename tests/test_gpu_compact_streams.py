"""Compactions of one context on several streams and beside replayed graphs, on the GPU: each moves rows of its own, none waits for what another has cleared."""
import numpy as np
import pytest
from oracle import tree_oracle as T
from pooled_amd.capi import PooledAttn
from test_gpu_tree_run import Graph

pytestmark = pytest.mark.gpu
SEQ, PARTS = 150000, [(5, 60000, 50000), (60000, 100000, 30000), (100000, 150000, 45000)]     # ranges of rows, and how many of each a call keeps


def context(kv_heads, q8):
    return PooledAttn(dict(n_heads=kv_heads, n_kv_heads=kv_heads, head_dim=128, n_rot=128, rope_theta=1e6, eps=1e-6, qk_norm=False, gate=False, kv_q8=q8), SEQ, n_layers=1, max_cols=1)


def filled(pa, rng):
    pa.layer_alloc(0)
    parts = []
    for w in range(4 if pa.cfg["kv_q8"] else 2):
        dt, per = pa._kv_part(w)
        parts.append(rng.integers(0, 100, (SEQ, pa.cfg["n_kv_heads"], per)).astype(dt))
        pa.kv_write(0, w, 0, parts[w])
    return parts


def lists(pa, rng, ranges):
    out = []
    for dst, end, n in ranges:
        rows = np.sort(rng.choice(end - dst, n, replace=False)) + dst
        out.append((dst, rows, pa.to_device(np.concatenate([[n], rows]).astype(np.uint32))))
    return out


def check(pa, parts, calls):
    for w, part in enumerate(parts):
        want = part
        for dst, rows, _ in calls:
            want = T.compact(want, dst, rows)
        assert np.array_equal(pa.kv_read(0, w, 0, SEQ), want), w


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("kv_heads", [1, 3])
def test_calls_on_three_streams(kv_heads, q8):
    """Enqueued in turn on different streams without a wait between them, on each a longer list and then a shorter one of the rows that are left."""
    rng, streams = np.random.default_rng(kv_heads), [Graph(), Graph(), Graph()]
    with context(kv_heads, q8) as pa:
        parts = filled(pa, rng)
        order = PARTS[1:2] + PARTS[:1] + PARTS[2:]                         # each range on one stream, twice
        calls = lists(pa, rng, order) + lists(pa, rng, [(dst, dst + n, n * 2 // 3) for dst, _, n in order])
        pa.sync()
        for i, (dst, rows, sel) in enumerate(calls):
            pa._chk(pa.L.pa_set_stream(pa.ctx, streams[i % 3].stream))
            pa.kv_compact(dst, sel, rows.size)
        for g in streams:
            pa._chk(pa.L.pa_set_stream(pa.ctx, g.stream))
            pa.sync()
        check(pa, parts, calls)
        pa._chk(pa.L.pa_set_stream(pa.ctx, None))
    for g in streams:
        g.close()


@pytest.mark.parametrize("q8", [False, True])
def test_replays_beside_eager_calls(q8):
    """A graph recorded behind an eager call of the same lengths, replayed on its stream while eager calls over other rows run on another."""
    rng, g, h = np.random.default_rng(7), Graph(), Graph()
    with context(2, q8) as pa:
        parts = filled(pa, rng)
        first, recorded = lists(pa, rng, [(100000, 150000, 49000)])[0], lists(pa, rng, PARTS[:1])[0]
        pa.kv_compact(first[0], first[2], first[1].size)
        pa.sync()
        pa._chk(pa.L.pa_set_stream(pa.ctx, g.stream))
        replay = g.record(lambda: pa.kv_compact(recorded[0], recorded[2], recorded[1].size))
        pa._chk(pa.L.pa_set_stream(pa.ctx, h.stream))
        for rep in range(3):
            for w, part in enumerate(parts):
                pa.kv_write(0, w, 0, part)
            pa.sync()
            eager = lists(pa, rng, PARTS[1:])
            g.hip.hipGraphLaunch(replay, g.stream)
            for dst, rows, sel in eager:
                pa.kv_compact(dst, sel, rows.size)
            g.hip.hipStreamSynchronize(g.stream)
            pa.sync()
            check(pa, parts, [recorded] + eager)
        pa._chk(pa.L.pa_set_stream(pa.ctx, None))
    g.close(); h.close()
