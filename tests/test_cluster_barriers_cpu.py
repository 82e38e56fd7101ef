"""The barriers of a cluster are executed by whole warps.

barrier.cluster.arrive and .wait in their aligned form are undefined for a warp that is not converged, and nothing converges it by itself
behind a branch that only some lanes take.  What that does depends on where the compiler joins the lanes again, and could be a cluster that
waits for good, so the sources are held to the rule instead of running them.
"""
import re

import pytest

from sharq_b200._build import CSRC
from tests.test_dependent_launch_cpu import _code

# what may stand directly ahead of a barrier: a convergence of the warp, another barrier, or a condition that all threads share
CONVERGED = re.compile(r"(__syncwarp\(\);|__syncthreads\(\);|ptx::cluster_(sync|arrive|wait)\(\);)\s*(if \((PAIR|split|a\.cluster > 1)\)\s*)?$")


@pytest.mark.parametrize("name", sorted(p.name for p in CSRC.glob("*.cu") if "cluster_sync()" in p.read_text()))
def test_full_barriers_follow_a_convergence(name):
    text = _code(CSRC / name)
    places = [m.start() for m in re.finditer(r"ptx::cluster_sync\(\)", text)]
    assert places
    for at in places:
        assert CONVERGED.search(text[:at]), text[max(0, at - 200):at + 20]


def test_the_files_that_have_them():
    assert {"paged_attention.cu", "weight_only.cu", "prepare.cu"} <= {p.name for p in CSRC.glob("*.cu") if "cluster_sync()" in p.read_text()}
