"""barrier.cluster.wait.aligned asks that all threads of a warp execute it together.  Where divergent code stands in front, the compiler as a
rule brings the warp together again, but nothing obliges it to: the source has to say so.  (What a warp that is not together does there
is undefined, so the source is read.)"""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ai-engine_b200", "csrc")


def test_the_wait_of_verification_brings_its_warp_together():
    with open(os.path.join(CSRC, "verify_drafts.cu")) as f:
        text = f.read()
    waits = [m.start() for m in re.finditer(r"barrier\.cluster\.wait\.aligned", text)]
    assert len(waits) == 1                              # all go through one function
    body = text[text.rindex("void cluster_wait()", 0, waits[0]):waits[0]]
    assert "__syncwarp();" in body
