"""Compaction of the caches to a list of rows (pa_kv_compact) on the GPU, bit for bit against the oracle."""
import numpy as np
import pytest
from oracle import tree_oracle as T
from pooled_amd.capi import PooledAttn, PaError, PA_ERR_INVALID
from helpers import SHAPES

pytestmark = pytest.mark.gpu


def filled(pa, layers, seed):
    """Random bits in every tensor of the layers; what is there, by (layer, tensor)."""
    rng = np.random.default_rng(seed)
    out = {}
    for l in layers:
        pa.layer_alloc(l)
        for w in range(4 if pa.cfg.get("kv_q8") else 2):
            dt, per = pa._kv_part(w)
            shape = (pa.max_seq, pa.cfg["n_kv_heads"], per)
            a = rng.standard_normal(shape).astype(np.float32) if dt == np.float32 else rng.integers(0, 256, shape + (np.dtype(dt).itemsize,), dtype=np.uint8).view(dt)[..., 0]
            pa.kv_write(l, w, 0, a)
            out[l, w] = a
    return out


def check(pa, was, dst, rows):
    for (l, w), a in was.items():
        got, want = pa.kv_read(l, w, 0, pa.max_seq), T.compact(a, dst, rows)
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8)), (l, w, dst, len(rows))
        was[l, w] = want


def ascending(rng, dst, end, n):
    return np.sort(rng.choice(np.arange(dst, end), n, replace=False))


SIZES = [(0, 40, 1), (3, 40, 0), (10, 34, 5), (0, 64, 64), (7, 200, 33), (50, 700, 400), (1, 3001, 1500), (0, 5000, 4999), (100, 9000, 1111), (5, 9000, 8800)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("dst,end,n", SIZES)
def test_lists(shape, dst, end, n, q8):
    rng = np.random.default_rng(dst + n)
    with PooledAttn(dict(SHAPES[shape], kv_q8=q8), end + 9, n_layers=3) as pa:
        was = filled(pa, (0, 2), n)                       # layer 1 has no cache
        print("compact", shape, q8, dst, end, n, flush=True)
        for rows in (ascending(rng, dst, end, n), ascending(rng, dst, end, n)):
            pa.run_kv_compact(dst, rows)
            check(pa, was, dst, rows)


def test_paths_that_stay_and_neighbours():
    """The identity, a shift by one row, and by one row behind a kept head: the rows that move next to themselves."""
    with PooledAttn(SHAPES["qwen36_moe"], 4000, n_layers=1) as pa:
        was = filled(pa, (0,), 1)
        for dst, rows in ((0, np.arange(4000)), (1500, np.arange(1500, 4000)), (0, np.arange(1, 4000)), (7, np.concatenate([np.arange(7, 900), np.arange(901, 4000)])), (0, np.arange(0, 4000, 2)),
                          (0, np.concatenate([np.arange(10), np.arange(3000, 3990)]))):
            pa.run_kv_compact(dst, rows)
            check(pa, was, dst, rows)


@pytest.mark.parametrize("q8", [False, True])
def test_long_lists(q8):
    """Many segments to a plane, kept rows of a tenth to nearly all, one call behind another."""
    with PooledAttn(dict(SHAPES["qwen38_27b"], kv_q8=q8), 40000, n_layers=2) as pa:
        was = filled(pa, (0, 1), 5)
        rng = np.random.default_rng(9)
        for dst, end, n in ((0, 40000, 36000), (4, 36000, 20000), (1000, 39000, 3800), (0, 40000, 39999)):
            rows = ascending(rng, dst, end, n)
            pa.run_kv_compact(dst, rows, max_rows=min(n + 17, 40000 - dst))
            check(pa, was, dst, rows)


def test_many_layers():
    """More tensors than one launch takes."""
    cfg = dict(n_heads=2, n_kv_heads=1, head_dim=128, n_rot=64, rope_theta=1e6, eps=1e-6, qk_norm=True, gate=False)
    for q8 in (False, True):
        with PooledAttn(dict(cfg, kv_q8=q8), 90, n_layers=150) as pa:
            was = filled(pa, range(150), 2)
            rows = ascending(np.random.default_rng(0), 30, 90, 21)
            pa.run_kv_compact(30, rows)
            check(pa, was, 30, rows)


def test_the_list_is_not_trusted():
    """A length word above max_rows is read as max_rows; rows outside the cache are clamped; in any order the rows outside [dst, dst + n) stay."""
    cfg = dict(SHAPES["qwen3_1p7b"])
    with PooledAttn(cfg, 600, n_layers=1) as pa:
        was = filled(pa, (0,), 3)
        sel = pa.to_device(np.concatenate([[0xFFFFFFFF], np.arange(40, 80)]).astype(np.uint32))
        pa.kv_compact(40, sel, 8); pa.sync()
        check(pa, was, 40, np.arange(40, 48))
        sel = pa.to_device(np.array([4, 100, 599, 600, 0xFFFFFFFF], np.uint32))
        pa.kv_compact(90, sel, 4); pa.sync()
        check(pa, was, 90, np.array([100, 599, 599, 599]))
        rng = np.random.default_rng(1)
        for n in (5, 300):
            before = {key: a.copy() for key, a in was.items()}
            pa.run_kv_compact(200, rng.integers(0, 600, n))
            for (l, w), a in before.items():
                got = pa.kv_read(l, w, 0, 600)
                keep = np.r_[0:200, 200 + n:600]
                assert np.array_equal(got[keep], a[keep])
                was[l, w] = got


def test_refusals():
    with PooledAttn(SHAPES["qwen36_moe"], 100, n_layers=1) as pa:
        sel = pa.to_device(np.zeros(120, np.uint32))
        with pytest.raises(PaError) as e:                 # no layer has a cache
            pa.kv_compact(0, sel, 4)
        assert e.value.code == PA_ERR_INVALID and "pa_layer_alloc" in str(e.value)
        pa.layer_alloc(0)
        for dst, ptr, most in ((0, None, 4), (0, sel.ptr + 2, 4), (0, sel.ptr, 0), (97, sel.ptr, 4), (0, sel.ptr, 101), (0xFFFFFFFF, sel.ptr, 2), (0, sel.ptr, 0xFFFFFFFF)):
            assert pa.L.pa_kv_compact(pa.ctx, dst, ptr, most) == PA_ERR_INVALID
            assert b"pa_kv_compact: " in pa.L.pa_last_error(pa.ctx)
        pa.kv_compact(0, sel, 100)                        # an empty list
        pa.sync()
        assert pa.L.pa_kv_compact(None, 0, sel.ptr, 1) == PA_ERR_INVALID
