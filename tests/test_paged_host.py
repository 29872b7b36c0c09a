"""What of the paged cache can be checked without a GPU."""
import os
import re


def test_waits_are_decided_by_whole_warps():
    """No wait of the attention kernel is branched on by a lane alone."""
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yapd_b200", "csrc",
                            "paged_attend.cu")).read()
    assert re.findall(r".*mbar_wait_bounded.*", src) == \
        ["  return __all_sync(~0u, yapd::mbar_wait_bounded(bar, parity, limit_ns));"]
