"""The waits of the shared-prefix attention kernel, checked in its source: what
would show on a GPU only as a kernel that never ends is not run there."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def source():
    """rv_prefix.cuh without comments."""
    with open(os.path.join(ROOT, "ramvamp_b200", "csrc", "rv_prefix.cuh")) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_every_wait_is_bounded(source):
    """No named barrier (a warp that gave up would never reach it), and
    mbarriers are waited on through the two bounded waits only."""
    assert not re.search(r"\b(bar|barrier)(\.cta)?\.(sync|red)", source)
    assert "__barrier_sync" not in source and "named_barrier" not in source
    assert len(re.findall(r"mbar_try_wait\(", source)) == 1
    wait1 = source[source.index("bool pfx_wait1("):source.index("bool pfx_wait(")]
    assert "mbar_try_wait(" in wait1 and "RV_WAIT_CYCLES" in wait1 and "return false" in wait1


def test_a_warp_leaves_its_role_as_one(source):
    """A role of whole warps asks for the failure flag by a vote: lanes that
    read it at different times would part, some to the CTA's barrier and some to
    the next vote.  Only the loads (one thread) and the code after the CTA's
    barrier, where nothing writes the flag, read it plainly."""
    loops = [x for x in source.splitlines() if re.search(r"\b(for|while) \(", x) and "s_fail" in x]
    assert len(loops) == 4
    plain = [x for x in loops if "pfx_failed(s_fail)" not in x]
    assert len(plain) == 1 and "pfx_feed(" in plain[0]  # the loads


def test_a_cta_that_gives_up_waits_for_what_is_in_flight(source):
    """A role may give up after the loads or the products have ended their own:
    the copies and products in flight are waited for behind the CTA's barrier,
    where every role's failure is known, and tensor memory is freed after that."""
    end = source[source.rindex("__syncthreads();", 0, source.index("if (*s_fail) {")):source.index("tc_dealloc(")]
    assert end.startswith("__syncthreads();") and "tc_commit(drained)" in end
    assert "mbar_wait_bounded(&kv_full" in end and "mbar_wait_bounded(drained, 0)" in end
    assert end.index("mbar_wait_bounded(drained, 0)") < end.rindex("__syncthreads();") < end.index("break;")
    assert source.count("tc_commit(drained)") == 1  # in no role
