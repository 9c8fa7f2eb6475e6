"""The cache and attention kernels must not use scratch memory: what does not fit
in registers would go through HBM in the loop over the tokens (a spilled tile kernel
took five times as long), and a private array indexed past its end would be an
access out of bounds.  Compiles their sources with the product's flags."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from test_kernel_resources import HIPCC, ROOT

CSRC = os.path.join(ROOT, "flashgann_amd", "csrc")


def _flags():
    mk = open(os.path.join(CSRC, "Makefile")).read()
    m = re.search(r"ATTENDFLAGS := (.*?)\n(?!\s)", mk, re.S)
    return [f for f in m.group(1).replace("\\\n", " ").replace("$(ARCH)", "gfx950").split() if f != "-fPIC"]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_no_scratch(tmp_path):
    assert "-packed-fp32-ops" in _flags()
    procs = []
    for name in ("fg_cache", "fg_attend", "fg_attend_tiles"):
        out = tmp_path / f"{name}.s"
        procs.append((name, out, subprocess.Popen([HIPCC, *_flags(), "--cuda-device-only", "-S", "-o", str(out), os.path.join(CSRC, name + ".hip")],
                                                  stdout=subprocess.DEVNULL, stderr=subprocess.PIPE, text=True)))
    seen = {}
    for name, out, p in procs:
        _, err = p.communicate(timeout=900)
        assert p.returncode == 0, (name, err[-2000:])
        asm = out.read_text()
        kernels = re.findall(r"^(_Z\w+):\s*; @", asm, re.M)
        sizes = [int(x) for x in re.findall(r"; ScratchSize: (\d+)", asm)]
        assert len(kernels) == len(sizes) > 0, name
        seen.update(zip(kernels, sizes))
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", asm), name
    assert len(seen) >= 2 + 16 + 8 + 8 and not {k: v for k, v in seen.items() if v}, {k: v for k, v in seen.items() if v}
