"""What the pair kernel's memory ordering rests on, read from its source: no run can show a missing order (the values come out
right for as long as the timing is kind), so the forms themselves are checked."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hearth_b200", "csrc")


def _body(text, start):
    """The braces' content of the function whose signature contains `start`."""
    at = text.index("{", text.index(start))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i]
    raise AssertionError(start)


def test_what_one_cta_hands_the_other_is_released_and_acquired_at_cluster_scope():
    text = open(os.path.join(CSRC, "i8_gemm.cu")).read()
    assert not re.search(r"mbarrier\.arrive\.relaxed", text)
    kernel = _body(text, "i8_pair_kernel(const I8Product")
    # every barrier of the pair kernel is signalled by the other CTA, by its copies or by the pair's MMAs
    waits = re.findall(r"\b(mbar_wait\w*|mbar_try\w*)\(", kernel)
    assert waits and set(waits) <= {"mbar_wait_pair", "mbar_try_cluster"}, waits
    assert ".acquire.cluster" in _body(text, "bool mbar_try_cluster(") and "mbar_try_cluster(" in _body(text, "bool mbar_wait_pair(")
    # the other CTA's half of a stage counts at the leader's barrier by itself: no thread passes its arrival on
    assert "cp.async.bulk.tensor" in _body(text, "void pair_load(") and "mbarrier::complete_tx::bytes.cta_group::2" in _body(text, "void pair_load(")
    remote = re.findall(r"mbar_arrive_remote\(([^)]*)\)", kernel)
    assert remote and all("empty" in r for r in remote), remote
