"""No-GPU checks of the delta-rule and experts entry points: struct layouts as a C compiler sees them, refusals that need no device, and the addon's table."""
import ctypes
import os
import shutil
import subprocess

import pytest
from pooled_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not installed")
@pytest.mark.parametrize("struct,mirror", [("pa_delta_config", "PaDeltaConfig"), ("pa_moe_config", "PaMoeConfig"), ("pa_moe_planes", "PaMoePlanes")])
def test_struct_layouts_match_header(tmp_path, struct, mirror):
    t = getattr(capi, mirror)
    fields = [f[0] for f in t._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pooled_attn.h"\nint main(void) { printf("%%zu", sizeof(%s)); %s return 0; }\n' % (
        struct, " ".join('printf(" %%zu", offsetof(%s, %s));' % (struct, f) for f in fields)))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(t)] + [getattr(t, f).offset for f in fields]


def test_null_handles_are_refused_without_a_device():
    L, null, out = capi.load(), None, ctypes.c_void_p()
    invalid = capi.PA_ERR_INVALID
    assert L.pa_delta_create(null, ctypes.byref(capi.PaDeltaConfig(1, 1, 64, 16, 0, 1, 0.0, 1e-6, 0)), ctypes.byref(out)) == invalid
    assert L.pa_moe_create(null, ctypes.byref(capi.PaMoeConfig(32, 32, 1, 1, 0, 0)), ctypes.byref(capi.PaMoePlanes()), ctypes.byref(out)) == invalid
    assert not out.value
    assert L.pa_delta_reset(null, null, 0) == invalid and L.pa_delta_read(null, null, 0, 0, null) == invalid and L.pa_delta_write(null, null, 0, 0, null) == invalid
    assert L.pa_delta_state_bytes(null, 0) == 0 and not L.pa_delta_state_ptr(null, 0, 0)
    assert L.pa_delta_glue(null, null, 0, null, 4, null, null, null, null, 1, null, null, 1, 1, null, 4, null, null, 1) == invalid
    assert L.pa_delta_decode(null, null, 0, null, 4, null, 4, null, 4, null, null, 1, 1, 1, null, 4, 0) == invalid
    assert L.pa_delta_prefill(null, null, 0, null, 4, null, 4, null, 4, null, null, 1, 1, null, 4, 0) == invalid
    assert L.pa_moe_layer(null, null, null, null, 4, 1, null, 4, null, null) == invalid


def test_addon_exports_when_built():
    addon = os.path.join(ROOT, "pooled_amd", "lib", "pooled_attn.node")
    if not (os.path.exists(addon) and shutil.which("node")):
        pytest.skip("addon or node missing")
    want = ["delta" + n for n in ("Create", "Destroy", "Reset", "Read", "Write", "StateBytes", "StatePtr", "Glue", "Decode", "Prefill")] + ["moe" + n for n in ("Create", "Destroy", "Layer")]
    js = "const a=require(%r); for (const w of %r) { if (typeof a[w] !== 'function') throw new Error('missing ' + w); let ok = 0; try { a[w](); } catch (e) { ok = 1; } if (!ok && !/StateBytes|StatePtr/.test(w)) throw new Error('no check of arguments: ' + w); }" % (addon, want)
    r = subprocess.run(["node", "-e", js], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
