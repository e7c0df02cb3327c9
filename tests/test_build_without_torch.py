"""The library stands without torch: only the layers' autograd nodes need its headers."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "ot-based-heterogeneous-multi-modal-fusion-embedding-for-ad-analysis-_amd", "csrc")


def _commands(**env):
    r = subprocess.run(["make", "-n", "-B", "-C", CSRC, "all"] + [f"{k}={v}" for k, v in env.items()], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    return r.stdout


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_make_without_torch_builds_the_library_alone():
    with_torch, without = _commands(), _commands(PYTHON="/bin/false")
    assert "-o ../otfuse/lib/_otf_layers.so" in with_torch and "otf_torch.cpp" in with_torch
    assert "otf_torch.cpp" not in without and "-o ../otfuse/lib/libotfuse.so" in without
