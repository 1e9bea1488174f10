"""No CTA leaves while a bulk copy into its shared memory is in flight, not even
after a bounded wait gave up.

Such a wait cannot be made to run out on a healthy GPU, so the rule is read
from the sources: the warp that issues the copies waits for its last ones
whether or not another warp has given up by then (that warp may give up later).
"""

import os
import re

import pytest
from conftest import ROOT


def _code(name):
    text = open(os.path.join(ROOT, "rotalabs_accel_b200", "csrc", name)).read()
    return re.sub(r"//[^\n]*", "", text)


def _kernel(code, name):
    start = re.search(name + r"\(const __grid_constant__", code).start()
    end = code.find("__global__", start)
    return code[start:end if end > 0 else None]


@pytest.mark.parametrize("name,kernel", [("rla_w8a8.cu", "w8a8_split_kernel"), ("rla_tc.cu", "w8a16_tc_kernel"),
                                         ("rla_stream.cu", "w8a16_stream_kernel")])
def test_the_producer_waits_for_its_last_copies(name, kernel):
    body = _kernel(_code(name), kernel)
    drain = re.search(r"if \(\*abort_flag\)[^;]*?for \(int \w+ = max\(0", body, re.S)
    assert drain is None, "the last copies are waited for only if a wait has given up already"
    assert re.search(r"for \(int \w+ = max\(0, (issued\w*) - \w+\); \w+ < \1; \+\+\w+\)\s*rla_mbar_wait\(&(?:sm\.)?full", body)


def test_the_pair_drains_when_both_ctas_are_through():
    body = _kernel(_code("rla_w8a8.cu"), "w8a8_pair_kernel")
    end = body[body.rindex("__syncthreads()"):]
    # both CTAs know both states, then the leader drains, then both leave
    order = [end.index(s) for s in ("sm.peer_abort_flag", "sm.peer_issued", "rla_cluster_sync()", "if (*abort_flag || sm.peer_abort_flag)",
                                    "w8a8_pair_drain", "rla_tmem2_dealloc")]
    assert order == sorted(order)
    assert end.count("rla_cluster_sync()") == 2
    assert end.rindex("rla_cluster_sync()") > end.index("w8a8_pair_drain")


@pytest.mark.parametrize("stages", [2, 6])
def test_the_pairs_bytes_add_up(stages):
    """The arithmetic of w8a8_pair_drain: whatever number of blocks each CTA had
    issued, every barrier that is waited for gets the bytes it expects."""
    code = _code("rla_w8a8.cu")
    drain = code[code.index("w8a8_pair_drain(W8PairShared"):]
    assert re.search(r"if \(i >= n0\) rla_mbar_arrive_expect_tx\(bar, 2 \* half\);\s*"
                     r"if \(i >= n1\) rla_mbar_complete_tx\(bar, 2 \* half\);", drain)
    for n0 in range(0, 20):
        for n1 in range(max(0, n0 - stages), n0 + stages + 1):
            last = max(n0, n1)
            for i in range(max(0, last - stages), last):
                expected = (4 if i < n0 else 0) + (2 if i >= n0 else 0)
                arrived = (2 if i < n0 else 0) + (2 if i < n1 else 0) + (2 if i >= n1 else 0)
                arrivals = (i < n0) + (i >= n0)
                assert expected == arrived and arrivals == 1, (n0, n1, i)
