"""Another rule of the kernels' sources that no run can show to be kept: lanes that a wait may have left apart leave a loop, or enter what all of them enter, by one vote."""
import os
import re

import pytest

from test_kernel_sources import SOURCES, _statements


@pytest.mark.parametrize("path", [p for p in SOURCES if os.path.basename(p) == "spg_fp8_layer.cu"], ids=os.path.basename)
def test_a_flag_that_others_raise_is_voted_on(path):
    """Behind a wait each lane may read the flag at a time of its own.  A branch on it, where whole warps go on to meet, is by __any_sync; behind a barrier of the whole CTA
    nobody raises it any more."""
    before, found = "", 0
    for statement in _statements(path):
        if re.search(r"\bif \(.*\*abort_flag", statement):
            found += 1
            assert "__any_sync" in statement or before == "__syncthreads()", statement
        before = statement
    assert found >= 4, found
