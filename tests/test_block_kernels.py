"""No-GPU check of what is built for the blocks beside attention: every kernel in the device code is one that the host side launches."""
import re
import shutil
import subprocess

import pytest
from pooled_amd import build

NAME = rb"_Z\d+pa_(?:moe|delta|fill)_\w*kernel\w*"


@pytest.mark.skipif(shutil.which("nm") is None, reason="nm not installed")
def test_every_kernel_is_launched_by_something():
    device = {n.decode() for n in re.findall(NAME, open(build.LIB, "rb").read())}
    host = {w for line in subprocess.run(["nm", build.LIB], capture_output=True, text=True, check=True).stdout.splitlines() for w in line.split()[-1:]}
    assert len(device) > 30
    assert not device - host, "built, but out of every call's reach: %s" % sorted(device - host)
