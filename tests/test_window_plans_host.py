"""Rows that the prompts' window kernel does again key by key are planned in the buffers of the jobs' plans: read from the source that this waits for the last reader of a plan.
(The warp that fills up blocks walks over whole ones without waiting for anything, so that the output of the last job may leave before it has read to that job's end.)"""
import os
import re

import llmdivedeep_b200


def test_plans_are_written_over_when_nobody_reads_them():
    with open(os.path.join(os.path.dirname(llmdivedeep_b200.__file__), "csrc", "window_prompt.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    last, again = text.index("drain(k - 1, e, true);"), text.index("PromptPlan& p = plans[qd];")
    assert re.search(r"if \(redos > 0 && ok\) ok = wait\(&plan_free\[\(k - 1\) % kWpPlans\], \(k - 1\) / kWpPlans\);", text[last:again])
    assert "ok && x < redo_jobs" in text[last:again]
