"""What one block of a pair hands to the other goes through barriers that order memory over the pair.

An mbarrier arrival or wait without semantics and scope orders the own block's threads only.  The order
shows in the source; nothing is run."""

from __future__ import annotations

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "adamw4bit_b200", "csrc")


def _source(name):
    return open(os.path.join(CSRC, name)).read()


def test_arrivals_at_the_other_block_name_their_scope():
    found = 0
    for name in os.listdir(CSRC):
        for op in re.findall(r'"[^"]*(mbarrier\.arrive\S*shared::cluster\S*)', _source(name)):
            found += 1
            assert re.match(r"mbarrier\.arrive\.(release|relaxed)\.cluster\.shared::cluster", op), (name, op)
    assert found


def test_values_of_the_second_block_are_acquired_over_the_pair():
    tc, wgrad = _source("aw4_tc.cuh"), _source("aw4_wgrad.cu")
    waits = re.findall(r'"\{ \.reg \.pred p; (mbarrier\.try_wait\S*)', tc)
    assert "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64" in waits
    # what is told to the first block is released, and the thread that issues the products acquires it
    tell = re.search(r"(\w+)\(in_first_block\(smem_addr\(&s\.ready\[buf\]\)\)\)", wgrad).group(1)
    arrive = re.search(tell + r"\(uint32_t cluster_bar\) \{\s*asm volatile\(\"(\S+)", tc).group(1)
    assert arrive.startswith("mbarrier.arrive.release.cluster")
    product = wgrad[wgrad.index("warp == kWgProduct) {"):wgrad.index("tc_mma_f16(tmem")]
    assert re.search(r"bar_wait<kWaitPair>\(smem_addr\(&s\.ready\[buf\]\)", product)
