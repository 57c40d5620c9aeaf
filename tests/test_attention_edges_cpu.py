"""What the attention kernels' sources have to keep where no run can show it."""

import os
import re

import numpy as np

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


def test_pairs_of_weights_on_the_multiply_add_pipes():
    """ex2_pair, restated in numpy with the constants of its source: 2^x to 3e-6 (its polynomial's 2.8e-6 and three roundings), 1 at 0, and
    nothing at all at -inf, whose polynomial and exponent have to cancel bit for bit."""
    text = source("attn_tc.cu")
    body = text[text.index("f2 ex2_pair(f2 x) {"):]
    body = body[:body.index("\n}\n")]
    lowest, = set(re.findall(r"fmaxf\(v\.[xy], (-[\d.]+)f\)", body))
    c4, c3 = map(float, re.search(r"f2 p = f2_fma\(f2_all\(([\d.]+)f\), f, f2_all\(([\d.]+)f\)\)", body).groups())
    c2, c1, c0 = map(float, re.findall(r"p = f2_fma\(p, f, f2_all\(([\d.]+)f\)\)", body))
    f32, fma = np.float32, lambda a, b, c: (a.astype(np.float64) * b + c).astype(np.float32)

    def ex2_pair(x):
        x, magic = np.fmax(x, f32(lowest)), f32(12582912.0)
        t = x + magic
        f = x + fma(t, -1.0, float(magic))
        p = np.full_like(f, f32(c4))
        for c in (c3, c2, c1, c0):
            p = fma(p, f, float(f32(c)))
        return (p.view(np.uint32) + (t.view(np.uint32) << np.uint32(23))).view(np.float32)

    x = np.concatenate([np.linspace(-125, 9, 400_001), np.linspace(-1, 1, 400_001)]).astype(f32)
    assert np.abs(ex2_pair(x) / np.exp2(x.astype(np.float64)) - 1).max() <= 3e-6
    small = ex2_pair(np.linspace(-140, -124, 400_001).astype(f32))
    assert (small >= 0).all() and (small <= f32(2.0 ** -124 * 1.001)).all()
    assert ex2_pair(np.array([-np.inf, -1e30, -127.0], f32)).tolist() == [0.0, 0.0, 0.0] and ex2_pair(np.zeros(1, f32)).tolist() == [1.0]
