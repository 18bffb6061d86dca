"""No-GPU checks of the drafted-tree calls: the oracle's pins, the mask helpers of the binding, the plan rule, the mask window that the kernel cuts out."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
from oracle import attn_oracle as O
from oracle import tree_oracle as T
from pooled_amd import capi
from helpers import SHAPES

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pooled_amd", "csrc")


def test_tree_attention_of_a_triangle_is_a_verify_block():
    cfg = SHAPES["qwen3_1p7b"]
    rng = np.random.default_rng(0)
    n, base = 5, 9
    q = rng.standard_normal((n, cfg["n_heads"], cfg["head_dim"]), dtype=np.float32)
    k, v = (rng.standard_normal((base + n, cfg["n_kv_heads"], cfg["head_dim"])).astype(np.float16).view(np.uint16) for _ in range(2))
    gate = rng.standard_normal(q.shape, dtype=np.float32)
    got = T.tree_attention(q, k.view(np.float16), v.view(np.float16), base, np.tril(np.ones((n, n), bool)), gate)[0]
    assert np.abs(got - O.attention(q, k, v, base, gate=gate)).max() < 1e-12


def test_tree_attention_by_hand():
    """Two heads of one kv head, head_dim 2, two drafted rows without a context: the first column sees itself, the second both, a third nothing."""
    q = np.array([[[1.0, 0.0], [0.0, 1.0]]] * 3)
    k = np.array([[[0.0, 0.0]], [[np.sqrt(2) * np.log(3.0), 0.0]], [[9.0, 9.0]]])
    v = np.array([[[1.0, -2.0]], [[5.0, 6.0]], [[7.0, 7.0]]])
    out, absolute, reach = T.tree_attention(q, k, v, 0, np.array([[1, 0, 0], [1, 1, 0], [0, 0, 0]], bool))
    assert np.allclose(out[0], [[1, -2], [1, -2]]) and not out[2].any()
    assert np.allclose(out[1], [[0.25 * 1 + 0.75 * 5, -0.25 * 2 + 0.75 * 6], [3, 2]])          # weights 1 : 3 and 1 : 1
    assert np.allclose(absolute[1, 1], [3, 4]) and np.isclose(reach[1, 0], np.log(3.0))


def test_glue_at_pins():
    cfg = SHAPES["qwen36_moe"]
    n, base = 4, 1000
    d = O.make_inputs(cfg, 0, n, 1)
    half = cfg["n_rot"] // 2
    args = (d["qraw"], d["kraw"], d["vraw"], d["qw"], d["kw"])
    line, ref = base + np.arange(n), O.glue_kv(*args, base, cfg)
    one = T.glue_at(*args, line[None], np.zeros(half, int), cfg)
    assert np.array_equal(one["q"], ref["q"]) and np.array_equal(one["gate"], ref["gate"]) and np.array_equal(O.f16_bits(one["k"]), ref["k16"]) and np.array_equal(O.f16_bits(one["v"]), ref["v16"])
    axis = np.arange(half) % 3
    assert np.array_equal(T.glue_at(*args, np.stack([line] * 3), axis, cfg)["q"], ref["q"])
    other = T.glue_at(*args, np.stack([line, line + 5, line]), axis, cfg)["q"]                  # the second axis moved: its pairs alone differ
    moved = np.any(other != ref["q"], axis=(0, 1))
    assert moved[1:half:3].all() and moved[half + 1:2 * half:3].all() and moved.sum() == 2 * len(range(1, half, 3))


def test_compact_row_by_row():
    rng = np.random.default_rng(2)
    cache = rng.standard_normal((40, 2, 3))
    rows = np.sort(rng.choice(np.arange(7, 40), 11, replace=False))
    want = cache.copy()
    for i, r in enumerate(rows):                    # ascending from dst on: in order, a row is read before it is overwritten
        want[7 + i] = want[r]
    assert np.array_equal(T.compact(cache, 7, rows), want)


def test_mask_helpers():
    seen = capi.tree_of_parents([-1, 0, 0, 1, -1, 4])
    assert seen.astype(int).tolist() == [[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 0, 1, 0, 0, 0], [1, 1, 0, 1, 0, 0], [0, 0, 0, 0, 1, 0], [0, 0, 0, 0, 1, 1]]
    assert capi.tree_mask(seen).tolist() == [[1], [3], [5], [11], [16], [48]]
    wide = np.zeros((70, 70), bool)
    wide[3, [0, 31, 32, 63, 64, 69]] = True
    assert capi.tree_mask(wide)[3].tolist() == [0x80000001, 0x80000001, 0x21] and not capi.tree_mask(wide)[4].any()
    with pytest.raises(ValueError):
        capi.tree_of_parents([-1, 1])


WINDOW = r"""
#include "tree_mask.h"
#include <cstdio>
#include <random>
int main() {
  std::mt19937 r(3);
  long seen = 0;
  for (int it = 0; it < 200000; it++) {
    const uint32_t n = 1 + r() % 140, words = (n + 31) / 32;
    uint32_t row[8];
    for (uint32_t w = 0; w < words; w++) row[w] = r();                 // bits from n on are set as well, words behind do not exist
    for (uint32_t w = words; w < 8; w++) row[w] = 0xdeadbeef;
    const int off = -31 + (int)(r() % (31 + (n + 31)));
    const uint32_t got = mask_window(row, off, n);
    for (int i = 0; i < 32; i++) {
      const int j = off + i;
      const uint32_t want = j < 0 ? 1u : j >= (int)n ? 0u : row[j / 32] >> (j % 32) & 1;
      if ((got >> i & 1) != want) { printf("n %u off %d bit %d\n", n, off, i); return 1; }
      seen += want;
    }
  }
  puts(seen > 1000000 ? "ok" : "too few");
}
"""


def test_mask_window(tmp_path):
    src, exe = tmp_path / "t.cc", tmp_path / "t"
    src.write_text(WINDOW)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC, str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def tree_rule(cfg, base, n, splits=0, most=0xffffffff):
    """(nb, waves, n_groups, group_rows, n_splits, split_tiles) of a call on a part of 256 CUs; no GPU needed."""
    c = capi.PaConfig(cfg["n_heads"], cfg["n_kv_heads"], cfg["head_dim"], cfg["n_rot"], cfg["rope_theta"], cfg["eps"], base + n, 1, n, capi.PA_FLAG_KV_Q8 if cfg.get("kv_q8") else 0)
    out = (ctypes.c_uint32 * 6)()
    u32 = ctypes.c_uint32
    assert capi.load().pa_rule_tree(ctypes.byref(c), ctypes.c_int(256), u32(base), u32(n), u32(splits), u32(most), out) == 0
    return tuple(out)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shape", sorted(SHAPES) + ["64 heads", "no groups"])
def test_plans_cover_rows_and_tiles(shape, q8):
    """Every stacked row is in one group that its workgroup's waves hold, every tile in one split, no group and no split is empty, and a limit on the splits is kept."""
    cfg = dict(SHAPES.get(shape) or dict(SHAPES["qwen3_1p7b"], n_heads=64 if shape == "64 heads" else 3, n_kv_heads=1 if shape == "64 heads" else 3), kv_q8=q8)
    G = cfg["n_heads"] // cfg["n_kv_heads"]
    for n in [1, 2, 3, 7, 8, 9, 16, 17, 24, 31, 33, 48, 63, 64, 65, 100, 128, 200, 333, 1000]:
        for base in [0, 1, 31, 32, 100, 1000, 4097, 20003, 65536, 500000]:
            for splits, most in [(0, 0xffffffff), (0, 5), (0, 0), (1, 0xffffffff), (7, 0xffffffff), (100000, 0xffffffff)]:
                nb, waves, groups, rows, ns, tiles = tree_rule(cfg, base, n, splits, most)
                assert rows <= 16 * nb * waves and (groups - 1) * rows < n * G <= groups * rows
                assert (ns - 1) * tiles * 32 < base + n <= ns * tiles * 32
                assert ns <= max(most, 1) and (not splits or ns <= splits)


def test_wait_states_behind_matrix_instructions(tmp_path):
    """As tests/test_wait_states.py has it for the chunked delta rule: on every path of the built kernels the hardware's wait states are kept."""
    from test_wait_states import NEEDED, disassembled, shortest
    kernels = {n: c for n, c in disassembled("attn_tree", tmp_path).items() if "pa_tree_kernel" in n}
    assert kernels
    for name, code in kernels.items():
        uses = shortest(code)
        assert len(uses) >= 8 and all(op in NEEDED for op, _, _ in uses), name
        low = min(uses, key=lambda u: u[1] - NEEDED[u[0]])
        assert low[1] >= NEEDED[low[0]], "%s: %d wait states behind %s in front of %s" % (name, low[1], low[0], low[2])


def test_every_kernel_is_launched_by_something():
    import re
    import shutil
    from pooled_amd import build
    if shutil.which("nm") is None:
        pytest.skip("nm not installed")
    device = {n.decode() for n in re.findall(rb"_Z\d+pa_(?:tree|glue_at|compact)_\w*kernel\w*", open(build.LIB, "rb").read())}
    host = {w for line in subprocess.run(["nm", build.LIB], capture_output=True, text=True, check=True).stdout.splitlines() for w in line.split()[-1:]}
    assert len(device) >= 6 and not device - host, sorted(device - host)
