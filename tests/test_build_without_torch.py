"""The C ABI library builds where torch or Python's headers are missing (JAX and C users); only the serving operators'
native front-end, a module over torch, needs them. Dry runs of make: nothing is compiled."""

import os
import subprocess
import sys

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "algebraic-extra_b200", "csrc")


def planned(python):
    r = subprocess.run(["make", "-C", CSRC, "-n", "-B", "all", f"PYTHON={python}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_all_without_torch_leaves_the_front_end_out():
    out = planned("false")
    assert "libalgx.so" in out and "algx_native.cc" not in out and "not built" in out


def test_all_with_torch_builds_everything():
    out = planned(sys.executable)
    assert "libalgx.so" in out and "algx_native.cc" in out and "not built" not in out
