"""Values read from tensor memory are used only behind a wait that names them (checked on the
sources: the compiler may move arithmetic across a wait that does not)."""
import glob
import os
import re

import pytest

from hayate_b200.build import CSRC

SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")))


def code(path):
    text = open(path).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_every_read_is_waited_for_by_name(path):
    text = code(path)
    assert not re.findall(r"tmem_wait_ld\s*\(\s*\)", text)
    for m in re.finditer(r"^\s*tmem_ld32\(([^;]+)\);", text, flags=re.M):
        value = m.group(1).rsplit(",", 1)[1].strip()
        rest = text[m.end():]
        wait = re.search(r"tmem_wait_ld\(\s*%s\s*\);" % re.escape(value), rest)
        assert wait, value
        # between the two: other reads and their waits alone
        between = rest[:wait.start()]
        assert not re.sub(r"tmem_(ld32|wait_ld)\([^;]+\);", "", between).strip(), between
