"""The library and the program build without torch, the binding for the interpreter that asks."""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

from conftest import ROOT


def commands(python):
    """What a build from nothing would run; nothing is run."""
    out = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "flashgann_amd", "csrc"), "all", f"PYTHON={python}"],
                         check=True, capture_output=True, text=True).stdout
    assert "-o " + os.path.join(ROOT, "flashgann_amd", "libflashgann.so") in out and "bin/gpu_flashgann" in out
    return out


def test_without_torch():
    """An interpreter that finds no torch (its site-packages left out), and none at all."""
    for python in (f"{sys.executable} -S -I", "/nonexistent/python"):
        assert "torch" not in commands(python)


def test_the_interpreter_that_asks():
    out = commands(sys.executable)
    assert "flashgann_amd/_attention" + sysconfig.get_config_var("EXT_SUFFIX") + " " in out
    assert f"$({sys.executable} -c" in out and "$(python3 -c" not in out


def test_the_binding_in_use_is_of_this_interpreter():
    from flashgann_amd import attention
    assert attention._attention.__file__.endswith("_attention" + sysconfig.get_config_var("EXT_SUFFIX"))
