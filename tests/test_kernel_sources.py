"""Rules of the kernels' sources that no run can show to be kept, read from the sources themselves."""
import glob
import os
import re

import pytest

from conftest import ROOT

SOURCES = sorted(glob.glob(os.path.join(ROOT, "spingalett_b200", "csrc", "cuda", "*.cu*")))


def _statements(path):
    """The file's statements without comments, a line's string literals left as they are."""
    with open(path) as f:
        text = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
    return [s.strip() for s in re.split(r"[;{}](?=[^\"]*(?:\"[^\"]*\"[^\"]*)*$)", text, flags=re.M) if s.strip()]


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_warps_meet_before_a_barrier_of_their_cluster(path):
    """The .aligned forms ask for all threads of a warp at once: behind a branch by lane, or a loop whose lanes end at different times, the
    warp has to meet first.  Each stands directly behind __syncwarp, or behind another such barrier."""
    before = ""
    for statement in _statements(path):
        if re.search(r"barrier\.cluster\.(arrive|wait)\S*\.aligned", statement):
            assert before == "__syncwarp()" or "barrier.cluster" in before, statement
        before = statement


def test_the_barriers_are_found():
    """(What the test above looks at is there.)"""
    found = [s for path in SOURCES for s in _statements(path) if "barrier.cluster" in s]
    assert len(found) >= 4, found
