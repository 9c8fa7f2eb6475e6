"""The batches of the tests of attention over selected pages run the kernels that they are
there for: tiles of 32 rows, of 16, and of 16 whose parts are joined."""
from __future__ import annotations

import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_which_kernel(gpu_available):
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "which_kernel.py")
    p = subprocess.run([sys.executable, at], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stderr[-2000:]
    names = json.loads(p.stdout.strip().splitlines()[-1])
    assert len(names) >= 16
    rows32, rows16, join = "fg_blocks_chunk_kernel", "fg_blocks_kernel", "fg_blocks_join_kernel"
    for name, kernels in names.items():
        if name.startswith("many"):
            assert kernels == [rows32], name
        else:
            assert kernels[0] == rows16 and set(kernels[1:]) <= {join}, name
    assert names["single tokens"] == [rows16] and names["one token, many pages"] == [rows16, join]
