"""What the attention kernels' sources have to keep where no run can show it."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "experiment_swa_kda_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def test_lists_in_shared_memory_end_before_copies_take_their_place():
    """The search for a part's length leaves its lists where the queries go; an ordinary access and a bulk copy to the same place are
    ordered by a fence of the asynchronous proxy and the barrier behind it."""
    text = source("attn_tc.cu")
    lists, setup = text.index("blocks_of = tiles_of"), text.index("mbar_init(bar_q")
    assert lists < text.index("fence_async_smem();", lists) < setup < text.index("__syncthreads();", setup)


def test_warps_agree_on_how_their_waits_ended():
    """A bounded wait that runs out in some lanes of a warp only must not part them: outside of the one lane that issues the products, every
    wait in the tensor-core kernel is the warp's."""
    text = source("attn_tc.cu")
    lane = text[text.index("if (t_begin < t_end && elect_one())"):text.index("} else if (warp == kLoadWarp) {")]
    waits = re.compile(r"(?<![\w.])wait\(bar")
    assert len(waits.findall(lane)) > 0 and len(waits.findall(text)) == len(waits.findall(lane))
    assert "__all_sync(0xffffffffu, wait(w, parity))" in text
