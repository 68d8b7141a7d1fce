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


@pytest.mark.parametrize("path", [p for p in SOURCES if not p.endswith("cache_common.cuh")], ids=os.path.basename)
def test_every_bounded_wait_is_of_a_whole_warp_or_of_one_lane(path):
    """A wait whose lanes' limits end apart leaves a warp incomplete in the shuffles and tensor-memory loads behind it:
    whole warps leave it by a vote (warp_wait), and only the sections of one lane wait alone (lane_wait)."""
    text = code(path)
    assert not re.search(r"\bmbar_(try_|test_)?wait\b", text)
    if "lane_wait" in text:  # the copying lane's section
        section = {"cache_tc.cu": r"warp == 0 && lane == 0\) \{(.*?)\} else if \(warp == 1",
                   "cache_weights.cu": r"lane == 0 && count > 0\) \{(.*?)\} else if \(warp == 1"}[os.path.basename(path)]
        assert re.search(section, text, re.S).group(1).count("lane_wait") == text.count("lane_wait")


def test_the_waits_of_whole_warps_are_votes():
    text = code(os.path.join(PKG, "csrc", "cache_common.cuh"))
    body = re.search(r"bool warp_wait\([^)]*\) \{(.*?)\n\}", text, re.S).group(1)
    assert "__all_sync(0xffffffffu" in body and "mbar_wait(bar, parity" in body
