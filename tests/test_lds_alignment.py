"""LDS whose size the launch gives begins behind a kernel's other LDS, at the alignment that its declaration has: pieces of it
are read 16 bytes at a time, so every such declaration asks for 16 bytes or more."""
import glob
import os
import re

import pytest

from tinybatch_amd.build import CSRC

DECLARED = re.compile(r"extern\s+__shared__\s+(?P<align>__align__\((?P<bytes>\d+)\)\s+)?(?P<rest>[^;]*);")
FILES = sorted(f for f in glob.glob(os.path.join(CSRC, "*")) if "extern __shared__" in open(f).read())


def test_there_are_such_declarations():
    assert any(f.endswith("tb_beam_state.hip") for f in FILES)


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_launch_sized_lds_is_aligned_to_16_bytes(path):
    found = list(DECLARED.finditer(open(path).read()))
    assert found
    for m in found:
        assert m["bytes"] and int(m["bytes"]) % 16 == 0, m.group(0)
