"""What is built again, and when."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "time-gan_amd", "csrc")


@pytest.mark.parametrize("changed", ["Makefile", "tgru_internal.h", os.path.join("..", "..", "include", "tgru.h")])
def test_every_object_depends_on_flags_and_headers(changed):
    """As if `changed` had just been edited: make would compile every source (nothing is compiled here)."""
    plan = subprocess.check_output(["make", "-n", "-W", changed, "-C", CSRC], text=True)
    sources = [f for f in os.listdir(CSRC) if f.endswith(".hip")]
    assert len(sources) > 10
    for f in sources:
        assert f" -c {f} " in plan, f


def test_build_compiles_where_built_libraries_are(monkeypatch):
    sys.path.insert(0, ROOT)
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(entry.subprocess, "check_call", lambda cmd, *a, **kw: calls.append(cmd))
    entry.build()
    assert any(c[0] == "make" and "-B" in c and CSRC in c for c in calls)
    assert any(c[-1].endswith(os.path.join("csrc_torch", "build.sh")) for c in calls)
