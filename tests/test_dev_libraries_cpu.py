"""The development libraries of scripts/dev are linked from every source of the package: the binding asks for all entries when it loads."""
import os
import re

import pytest

from dun_amd.build import SOURCES

DEV = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scripts", "dev")


@pytest.mark.parametrize("script", ["build_exp_lib.sh", "build_prof_lib.sh"])
def test_every_source_is_linked(script):
    with open(os.path.join(DEV, script)) as f:
        text = f.read()
    copied = re.search(r"for f in ([a-z0-9 ]+);", text).group(1).split()
    compiled = re.findall(r"-c dun_amd/csrc/([a-z0-9]+)\.hip", text)
    assert sorted(copied + compiled) == sorted(s[:-len(".hip")] for s in SOURCES)


def test_a_change_of_the_flags_rebuilds_every_object(monkeypatch):
    """Objects that were compiled with other flags than build.py's are not linked into the library."""
    from dun_amd import build
    ran = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: (ran.append(cmd), build.subprocess.CompletedProcess(cmd, 0, "", ""))[1])
    newest = [os.path.abspath(build.__file__)]
    monkeypatch.setattr(build.os.path, "exists", lambda p: True)
    monkeypatch.setattr(build.os.path, "getmtime", lambda p: 2.0 if os.path.abspath(p) in newest else 1.0)
    build.build_library()
    compiled = {os.path.basename(c[c.index("-c") + 1]) for c in ran if "-c" in c}
    assert compiled == set(SOURCES)
    assert all("-packed-fp32-ops" in c for c in ran if "-c" in c)


def test_the_timing_library_is_compiled_like_the_package():
    with open(os.path.join(os.path.dirname(os.path.dirname(DEV)), "scripts", "gemm_phases.py")) as f:
        assert "B.FLAGS" in f.read()
