"""What the CUDA sources must state where no run can show it: the scope of signals between CTAs."""

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "telmo_b200", "csrc")


def sources():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*")) + glob.glob(os.path.join(CSRC, "*.h"))):
        with open(path) as f:
            yield os.path.basename(path), f.read()


def test_arrivals_on_another_cta_name_the_cluster_scope():
    """An arrival without a scope orders memory within its own CTA alone. (A product's commit, which tracks
    asynchronous operations, has no such choice.)"""
    found = 0
    for name, text in sources():
        for op in re.findall(r"mbarrier\.arrive[\w.:]*", text):
            if ".shared::cluster" in op and "::arrive::" not in op:
                found += 1
                assert re.search(r"\.(release|relaxed)\.cluster\b", op), (name, op)
    assert found >= 2


def test_a_pair_s_barriers_are_waited_for_at_cluster_scope():
    """Those that the other CTA signals in the tiles of the 4-bit product."""
    text = dict(sources())["q4_gemm.cu"]
    for bar in ("full[st.at]", "empty[st.at]", "acc_full[ab.at]", "acc_empty[acc.at]"):
        waits = re.findall(r"(\w+)(?:<[^<>]*>)?\(&" + re.escape(bar) + r", \w+\.phase", text)
        assert waits and set(waits) == {"wait_for_pair"}, (bar, waits)
