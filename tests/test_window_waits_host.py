"""The window kernels promise that a wait which runs out ends the call with a status.  A hardware barrier has no limit, so it may stand only where every warp that it counts
comes, whatever became of that warp's waits: read from the sources."""
import os
import re

import llmdivedeep_b200

CSRC = os.path.join(os.path.dirname(llmdivedeep_b200.__file__), "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_the_prompts_kernel_has_no_barrier_among_some_of_its_warps():
    assert "named_bar_sync" not in source("window_prompt.cu")


def test_barriers_behind_a_condition_are_reached_by_all_of_a_quadrant():
    """In the records' kernel the rows to be done again stand between two barriers of a quadrant's four warps: whether one of these has given up is agreed on at the barrier
    before, which none of them passes by."""
    text = source("window_mla.cu")
    again = text.index("if (again)")
    before = text[text.rindex("named_bar_sync(3 + qd, 128);", 0, again):again]
    said = text[:text.index(before)]
    assert "lost_s[qd] = 1;" in said and re.search(r"ok = lost_s\[qd\] == 0;", before)
    assert re.search(r"if \(ok\) \{.*again = __ballot_sync", before, re.S)
    # from the last softmax block to that barrier nothing leaves
    tail = said[said.index("if (ok) ok = mla_wait(o_final"):]
    assert not re.search(r"\b(return|break|continue)\b", tail)


def test_what_the_other_sm_stores_is_waited_for_at_the_clusters_scope():
    for name in ("window_prompt.cu", "window_mla.cu"):
        text = source(name)
        assert "wait_scores(&recv_full[warp]" in text and not re.search(r"\b(mla_)?wait\(&recv_full", text)
    assert "mbar_wait_warp<4, true>" in source("window_mla.cuh") and "try_wait.parity.acquire.cluster" in source("dsa_common.cuh")
