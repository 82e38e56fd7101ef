"""A wait inside ops.prompt_attention that runs out: reported, and the GPU goes on as before."""
import pytest
import torch

from sharq_b200 import ops
from tests.gpu_util import call
from tests.test_prompt_attention_gpu import check, ends, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_a_wait_that_runs_out_is_reported(dim):
    """The one sequence with rows is behind 200000 empty ones, so that the search for it takes more than a million cycles, and the limit is a tenth of one: every
    other warp has given up when the copies for it are issued, which the block has to wait for all the same."""
    lengths = [0] * 200000 + [100]
    q, k, v = inputs(lengths, lengths, 4, 2, dim, 3)
    at = ends(lengths)
    want = ops.prompt_attention(q, k, v, at, window=30, sinks=2)
    check(want, q, k, v, [100], [100], 30, 2)
    ops.check_device_errors()
    try:
        call("sharq_set_wait_limit_cycles", 100_000)
        for _ in range(3):
            ops.prompt_attention(q, k, v, at, window=30, sinks=2)
            with pytest.raises(RuntimeError, match="a wait ran out"):
                ops.check_device_errors()
    finally:
        call("sharq_set_wait_limit_cycles", 0)
    for _ in range(3):
        assert torch.equal(ops.prompt_attention(q, k, v, at, window=30, sinks=2), want)
    ops.check_device_errors()


def test_a_limit_that_nothing_reaches_changes_nothing():
    lengths = [700, 90, 1200]
    q, k, v = inputs(lengths, lengths, 8, 2, 128, 4)
    want = ops.prompt_attention(q, k, v, ends(lengths), window=300, sinks=4)
    try:
        for cycles in (100_000_000, 10 ** 15):  # longer than the default is the default
            call("sharq_set_wait_limit_cycles", cycles)
            assert torch.equal(ops.prompt_attention(q, k, v, ends(lengths), window=300, sinks=4), want)
    finally:
        call("sharq_set_wait_limit_cycles", 0)
    ops.check_device_errors()
