"""A kernel of the decode step whose wait for a copy runs out leaves nothing behind that still writes.

A copy that lands late would write into the shared memory of whichever CTA is there by then, and a barrier that is armed again while its
copy is on its way counts wrongly.  Making a copy late needs a GPU that stalls, so the sources are held to the rule instead: a lane whose
wait has failed waits (with a limit of its own) for all that is on its way, and the lane that copies requests nothing more.
"""
import re

import pytest

from sharq_b200._build import CSRC
from tests.test_dependent_launch_cpu import _block, _code


@pytest.mark.parametrize("name,lost,stages", [("paged_attention.cu", r"\(bad_stages & kLost\)", "kStages"),
                                              ("weight_only.cu", r"\(phases & kWoLost\)", "kWoStages")])
def test_a_wait_that_ran_out(name, lost, stages):
    code = _code(CSRC / name)
    assert code.count("mbar_wait(") == 1
    at = code.rindex("if (", 0, code.index("mbar_wait("))
    assert re.match(rf"if \({lost} == 0 && !ptx::mbar_wait\(", code[at:])
    given_up = _block(code, at)
    drain = re.search(rf"for \(int i = 0; i < {stages}; \+\+i\) ptx::mbar_drain\(bars \+ i, \(phases >> i\) & 1\);", given_up)
    assert drain and drain.start() < given_up.index("*gave_up = 1")
    assert re.search(r"(bad_stages \|= kLost|phases \|= kWoLost);", given_up)
    # the one lane that arms a barrier and issues copies does so only while the warp has lost nothing
    assert code.count("mbar_arrive_expect_tx(") == 1
    ahead = code[:code.index("mbar_arrive_expect_tx(")]
    assert re.search(rf"chosen (=|&&)[^;{{]*{lost} == 0[^;{{]*(;|\{{)\s*(if \(chosen\) |[^}}]*)ptx::$", ahead)


def test_the_second_wait_is_bounded_too():
    code = _code(CSRC / "sm100_ptx.cuh")
    assert "clock64() - start <= kWaitLimitCycles" in _block(code, code.index("void mbar_drain("))


def test_products_without_their_weight_are_nan():
    """Every sum that a CTA takes of its warps' parts behind a wait that ran out, whether it goes out or to the other CTAs of a cluster."""
    code = _code(CSRC / "weight_only.cu")
    at = code.index("const bool lost = *gave_up != 0;")
    assert "__syncthreads();" in code[code.rindex("}", 0, at):at]  # behind the warps' last wait
    sums = _block(code, code.index("for (int i = first + threadIdx.x; i < count;", at))
    poison = sums.index("if (lost) y.x = y.y = y.z = y.w = __int_as_float(0x7fffffff);")
    assert sums.rindex("add(y, v[s])") < poison < sums.index("finish(i, y)") and poison < sums.index("sum_of[i] = y")


def test_attention_behind_a_lost_tile_is_nan():
    """Every item that the lane takes part in from then on, finished or left as a part, by the sum of its probabilities."""
    code = _code(CSRC / "paged_attention.cu")
    at = code.index("const float lost = (bad_stages & kLost) != 0 ? __int_as_float(0x7fffffff) : 0.0f;")
    tiles, added = code.index("for (int tile = at.tile; tile < at.end; ++tile)"), code.index("l[n][j] += lost;", at)
    assert tiles + len(_block(code, tiles)) <= at
    assert code.index("l[n][j] += __shfl_xor_sync(", at) > added
    assert added < code.index("__fdividef(kFp8 ? c.v_scale[kv] : 1.0f, l[n][j])") and added < code.index("make_float4(m[n][0], l[n][0], m[n][1], l[n][1])")
