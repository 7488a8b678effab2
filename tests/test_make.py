"""What `make` builds for whom, from its dry run."""
import subprocess
import sys
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "scmiac_amd" / "csrc"


def _plan(python):
    done = subprocess.run(["make", "-B", "-n", "-C", str(CSRC), f"PYTHON={python}"], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    return done.stdout


def test_c_callers_need_no_torch(tmp_path):
    """Without torch, without Python headers and without Python, the C library is what `make` builds."""
    bare = tmp_path / "python-without-torch"
    bare.write_text(f'#!/bin/sh\nexec "{sys.executable}" -S "$@"\n')      # -S: no site-packages
    bare.chmod(0o755)
    for python in (bare, "/bin/false"):
        plan = _plan(python)
        assert "-o libscmiac_hip.so" in plan and "-o ../_torch_ops.so" not in plan and "not built" in plan


def test_with_torch_both_are_built():
    plan = _plan(sys.executable)
    assert "-o libscmiac_hip.so" in plan and "-o ../_torch_ops.so" in plan
