"""The bounded waits of the prompt kernel's whole-warp roles end for all lanes of a warp alike (CPU, by the source).

A lane that leaves a role alone would be missing from the next full-mask shuffle, vote or TMEM instruction of its warp,
which then need not end: the wait's bound would bound nothing. So in those roles a lane never acts on a wait of its own."""
import re

from conftest import ROOT

SOURCE = re.sub(r"//[^\n]*", "", (ROOT / "slotstream-spark_b200" / "csrc" / "paged_prefill.cu").read_text())
LONE = re.compile(r"(?<!\w)(?:wait|ready)\(")


def _roles():
    body = SOURCE[SOURCE.index("k_prefill(const __grid_constant__"):]
    copies, softmax = body.index("} else if (warp >= PROD) {"), body.index("const int t = warp >> 2")
    end = body.index("__syncthreads();", softmax)
    return body[copies:softmax], body[softmax:end]


def test_softmax_warps_wait_together():
    softmax = _roles()[1]
    assert not LONE.search(softmax) and softmax.count("warp_wait(") == 3
    assert re.findall(r"next_unit\(u, (\w+)", softmax) == ["WholeWarp"]


def test_copying_warps_wait_together():
    copies = _roles()[0]
    cut = copies.rindex("cp_async_wait_all();")
    work, drain = copies[:cut], copies[cut:]
    assert "_sync(" not in drain                       # after the last warp-wide instruction lanes may part
    hand_out = re.search(r"auto give_unit = \[&\] \{.*?\n    \};", work, re.S)
    rest = work[:hand_out.start()] + work[hand_out.end():]
    assert len(re.findall(r"give_unit\(\)", rest)) == len(re.findall(r"__all_sync\(0xFFFFFFFFu, give_unit\(\)\)", rest)) == 2
    voted = re.sub(r"__all_sync\(0xFFFFFFFFu, (?:ready|give_unit)\(", "", rest)
    assert not LONE.search(voted)
    assert re.findall(r"next_unit\(u, (\w+)", rest) == ["WholeWarp"]


def test_the_votes_are_there():
    assert re.search(r"bool warp_wait\([^)]*\) \{ return __all_sync\(0xFFFFFFFFu, wait\(bar, parity\)\); \}", SOURCE)
    assert re.search(r"by_warp\.value \? warp_wait\(u_full", SOURCE)
