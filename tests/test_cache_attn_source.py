"""Rules of the session-cache kernels that no run can show to be kept."""

import glob
import os
import re

import pytest

from conftest import PKG

SOURCES = sorted(glob.glob(os.path.join(PKG, "csrc", "cache_*.cu*")))


def code(path):
    """A source without its comments."""
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)


def test_the_sources_are_found():
    assert {os.path.basename(p) for p in SOURCES} >= {"cache_common.cuh", "cache_tc.cuh", "cache_tc.cu", "cache_decode.cu",
                                                      "cache_weights.cu", "cache_evict.cu", "cache_ops.cu"}


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_no_collective_of_a_guessed_set_of_lanes(path):
    """__activemask() says which lanes are together now, not which reach the next collective: a warp whose lanes the
    compiler has parted would wait in it with masks that disagree, without a bound."""
    assert "__activemask" not in code(path)
