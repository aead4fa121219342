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
