"""What is compiled again when the rules of the build change."""
import os
import shutil
import subprocess

import pytest

import tsc_hip
from test_kernel_resources import CSRC


def dry_run(*more):
    return subprocess.run(["make", "-n", "-C", CSRC, *more], check=True, capture_output=True, text=True).stdout


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_every_object_is_made_again_after_a_change_of_the_rules_or_a_header():
    sources = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
    headers = sorted(f for f in os.listdir(CSRC) if f.endswith(".h"))
    assert len(sources) >= 8 and headers
    for changed in ["Makefile", *headers]:
        out = dry_run("-W", changed)
        assert all(f"-c {s} " in out for s in sources), changed
        assert "-shared" in out


@pytest.mark.skipif(not os.path.exists(tsc_hip.library_path()), reason="libtsc_hip.so not built")
def test_build_compiles_what_is_there_already(monkeypatch):
    import __graft_entry__

    calls = []
    monkeypatch.setattr(__graft_entry__.subprocess, "run", lambda cmd, **kw: calls.append(cmd))
    __graft_entry__.build()
    assert len(calls) == 1 and "-B" in calls[0] and CSRC in calls[0]
