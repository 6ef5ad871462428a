"""How the one-kernel int8 expert layer takes over codes of h that other CTAs have written, read from the source: a wrong order cannot be shown by
running it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-scaler_b200", "csrc")


def test_flags_that_one_lane_has_seen_are_ordered_before_another_lanes_copies():
    """Each lane acquires a flag of its own and one elected lane issues the copies: the vote between them tells it the flags' values, but only a warp
    barrier orders its accesses behind theirs, and the fence between the proxies has to come behind that."""
    with open(os.path.join(CSRC, "moe_i8.cu")) as f:
        body = re.sub(r"//[^\n]*", "", f.read()).split("int wait_flags(")[1].split("\n}\n")[0]
    vote, fence = body.index("__ballot_sync("), body.index("fence.proxy.async")
    assert body.index("ld.acquire.gpu") < vote < fence
    assert "__syncwarp();" in body[vote:fence]
