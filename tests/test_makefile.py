"""The C library builds without Python and torch: `make lib`."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gat_amd", "csrc")


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_the_library_alone_asks_no_python(tmp_path):
    """a dry run with an interpreter that records any call of it"""
    trap = tmp_path / "python"
    trap.write_text(f"#!/bin/sh\ntouch {tmp_path}/called\nexit 1\n")
    trap.chmod(0o755)
    run = lambda target: subprocess.run(["make", "-n", "-B", "-C", CSRC, target, f"PYTHON={trap}"], capture_output=True, text=True)
    r = run("lib")
    assert r.returncode == 0 and "libgat_mi355.so" in r.stdout and "torch" not in r.stdout.replace("torch_dense", "")
    assert not (tmp_path / "called").exists()
    r = run("all")
    assert "_torch_dense.so" in r.stdout and (tmp_path / "called").exists()
