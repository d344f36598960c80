"""Every interleaving of the rows kernel's exchange of partial sums (``csrc/fp4_gemm_rows.cu``).

The CTAs of a cluster split K; row group g of A is added by the CTA of rank g % C, and the others send it
their sums. From 32 columns on the sums leave by ``cp.async.bulk`` out of the sender's shared memory, which a copy
reads until its bytes are counted at the receiver; below that by ``st.async``, whose values have left the sender when
it is issued. A CTA may leave only when no copy that reads or writes its memory is on its way.

The model runs, for each CTA, the steps that the kernel's source has, in the source's order, and completes copies at
any time. It asserts that no CTA leaves too early and that no state is stuck.
"""

from __future__ import annotations

import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ash-quant-kernels_b200", "csrc", "fp4_gemm_rows.cu")


def _way_out(staged):
    """The steps from the copies on, as the kernel has them for the staged or the st.async form."""
    text = open(SOURCE).read()
    text = re.sub(r"//[^\n]*", "", text[text.index("bulk_to_cluster(map_rank(to, owner)") :])
    text = text[: text.index("std::atomic<int> g_cluster")]
    steps = ["send"]
    pattern = r"(?:if \((!?)L::kStaged\) (\{[^}]*\}|[^;{]*;))|(mbar_wait_cluster\(received)|(cluster_arrive\(\);)|(cluster_wait\(\);)"
    for m in re.finditer(pattern, text):
        if m.group(2) is not None:
            if (m.group(1) == "!") != staged and "cluster_arrive();" in m.group(2):
                steps.append("arrive")
            assert "cluster_wait" not in m.group(2) and "received" not in m.group(2)
        else:
            steps.append("receive" if m.group(3) else "arrive" if m.group(4) else "wait")
    assert sorted(steps) == ["arrive", "receive", "send", "wait"], steps
    return steps + ["leave"]


def _explore(C, groups, steps, reads_sender):
    owners = [g % C for g in range(groups)]
    copies = [(src, dst) for dst in owners for src in range(C) if src != dst]
    expected = [sum(d == r for _, d in copies) for r in range(C)]
    init = ((0,) * C, (), (0,) * C)  # program counters, copies on their way, copies landed at each CTA
    seen, stack = {init}, [init]
    finished = False
    while stack:
        pcs, flying, landed = stack.pop()
        succ = []
        for i, (_, dst) in enumerate(flying):
            if i and flying[i] == flying[i - 1]:
                continue
            succ.append((pcs, flying[:i] + flying[i + 1 :], landed[:dst] + (landed[dst] + 1,) + landed[dst + 1 :]))
        arrived = sum(pc > steps.index("arrive") for pc in pcs)
        for r, pc in enumerate(pcs):
            if pc == len(steps):
                continue
            step, out = steps[pc], flying
            if step == "receive" and expected[r] and landed[r] < expected[r]:
                continue
            if step == "wait" and arrived < C:
                continue
            if step == "send":
                out = tuple(sorted(flying + tuple(c for c in copies if c[0] == r)))
            if step == "leave":
                assert not any(dst == r for _, dst in flying), f"CTA {r} left while a copy wrote into it"
                assert not (reads_sender and any(src == r for src, _ in flying)), f"CTA {r} left while a copy read its memory"
            succ.append((pcs[:r] + (pc + 1,) + pcs[r + 1 :], out, landed))
        if not succ:
            assert all(pc == len(steps) for pc in pcs), f"stuck at {pcs}"
            finished = True
        for s in succ:
            if s not in seen:
                seen.add(s)
                stack.append(s)
    assert finished


CASES = [(2, 1), (2, 2), (2, 3), (3, 1), (3, 2), (3, 3), (4, 1), (4, 2)]  # CTAs, groups: some own none


@pytest.mark.parametrize("C,groups", CASES)
@pytest.mark.parametrize("staged", [True, False], ids=["bulk", "st.async"])
def test_no_cta_leaves_early(C, groups, staged):
    _explore(C, groups, _way_out(staged), reads_sender=staged)


def test_the_model_sees_a_sender_that_leaves_early():
    with pytest.raises(AssertionError, match="read its memory"):
        _explore(3, 2, ["send", "arrive", "receive", "wait", "leave"], reads_sender=True)
