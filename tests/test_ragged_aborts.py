"""What the ragged attention kernels do after a bounded wait has run out, without a
GPU: the warps of a CTA leave together."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-vl_b200", "csrc")


def test_a_warp_reads_the_abort_flag_with_one_vote():
    """The flag is set by other warps at any time, so lanes that read it for
    themselves may part, and the rest of the warp then waits for them in a shuffle."""
    src = open(os.path.join(CSRC, "ragged_prefill.cu")).read()
    reads = [m.start() for m in re.finditer(r"\*abort_flag(?!\s*=[^=])", src)
             if not src[:m.start()].endswith("volatile int")]
    assert reads
    for at in reads:
        line = src[src.rfind("\n", 0, at) + 1:src.find("\n", at)]
        assert src[:at].endswith("__any_sync(0xffffffffu, "), line.strip()
