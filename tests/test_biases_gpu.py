"""Many biases on a token in ops.adjust_logits."""
import math

import pytest
import torch

from sharq_b200 import ops
from tests.test_logit_rules_gpu import case, check, rules64

pytestmark = pytest.mark.gpu


def several(vocab, n, of, seed):
    """n biases on `of` tokens each, in random order, whole numbers, so that 64 bits hold every sum of them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.arange(n, device="cuda") % (n // of)
    ids = (ids * 7919 % vocab)[torch.randperm(n, generator=g, device="cuda")].int()
    return torch.tensor([0, n], dtype=torch.int32, device="cuda"), ids, torch.randint(-9, 10, (n,), generator=g, device="cuda").float()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,n,of", [(1, 77, 77), (40, 900, 30), (33, 31, 1), (5000, 12000, 3), (32000, 2000, 2000), (152064, 40000, 2), (128256, 50000, 500)])
def test_sums_of_biases(vocab, n, of, dtype):
    logits, rules = case(1, vocab, 50, n, dtype)
    rules["bias"] = several(vocab, n, of, 1)
    got = ops.adjust_logits(logits, **rules)
    check(logits, got, rules64(logits, **rules))
    kept = logits.clone()
    assert torch.equal(ops.adjust_logits(logits, **rules), got) and torch.equal(logits, kept)
    assert torch.equal(ops.adjust_logits(logits, out=logits, **rules), got)
    ops.check_device_errors()


def test_a_bias_of_minus_zero_and_of_what_is_not_finite():
    """Sums as in the list's order: -0 leaves a zero's sign, infinities of both signs are NaN."""
    ids = [1, 2, 1, 3, 2, 3, 4, 4, 1000, -5, 5]
    values = [-0.0, math.inf, -0.0, math.inf, -math.inf, 5.0, math.nan, 1.0, 7.0, 7.0, math.inf]
    logits = torch.zeros(1, 40, device="cuda")
    logits[0, :2] = -0.0
    bias = tuple(torch.tensor(x, dtype=t, device="cuda") for x, t in (([0, 11], torch.int32), (ids, torch.int32), (values, torch.float32)))
    got = ops.adjust_logits(logits, bias=bias)[0].tolist()
    assert got[1] == 0 and math.copysign(1, got[1]) == -1 and math.copysign(1, got[0]) == -1
    assert math.isnan(got[2]) and got[3] == math.inf and math.isnan(got[4]) and got[5] == math.inf and got[6:] == [0.0] * 34
    with pytest.raises(RuntimeError, match="adjust_logits"):
        ops.check_device_errors()


@pytest.mark.parametrize("of", [2, 100000])
def test_the_time_grows_with_the_biases_not_with_their_square(of):
    """200000 biases, half of them on tokens that have several: linear, they take a fraction of a millisecond.  By comparing every one with every other
    they took a second; the bound lies between, far from both."""
    logits, _ = case(1, 128256, 1, 3)
    bias = several(4096, 200000, of, 2)
    bias[1][:100000] = torch.arange(20000, 120000, device="cuda").int()  # ahead of them as many that are alone
    times = []
    for _ in range(3):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        got = ops.adjust_logits(logits, bias=bias)
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    check(logits, got, rules64(logits, bias=bias))
    assert min(times) < 10, times
