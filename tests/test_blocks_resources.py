"""The kernels over selected pages and of eviction use no scratch memory and no packed
32-bit arithmetic, as the other cache kernels; compiled with the product's flags."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from test_attention_resources import CSRC, _flags
from test_kernel_resources import HIPCC


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_no_scratch(tmp_path):
    procs = []
    for name in ("fg_blocks", "fg_attend_blocks", "fg_evict"):
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
    # bounds, selection (five forms), rows, joins, chunks up to dim 128; weights; choosing (three), filling, shifting
    assert len(seen) == 8 + 40 + 8 + 8 + 6 + 8 + 3 + 2
    assert not {k: v for k, v in seen.items() if v}, {k: v for k, v in seen.items() if v}
