"""ops.prompt_attention at the edges of its contract: rows that belong to no sequence, keys that are not there, outputs over inputs, scores that are not finite."""
import math

import pytest
import torch

from sharq_b200 import ops
from tests.test_prompt_attention_gpu import bound, check, definition64, ends, inputs

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def leave_nan(like):
    """What the allocator hands out next, for tensors of that size, holds NaN."""
    torch.cuda.synchronize()
    held = [torch.full_like(like, math.nan) for _ in range(50)]
    torch.cuda.synchronize()
    del held


def accepted(at, rows):
    """The sequences that have rows: not those that go back, begin below an earlier beginning, or leave the rows."""
    reached, good = -1, []
    for a, b in zip(at, at[1:]):
        if a <= rows:
            reached = max(reached, a)
        if reached <= a <= b <= rows and a >= 0:
            good.append((a, b))
    return good


@pytest.mark.parametrize("at", [[0, 60, 50, 180], [0, 60, -2 ** 31, 180], [0, 2 ** 31 - 1, 110, 180], [-1, 60, 110, 180], [0, 60, 110, 181], [0, 100, 60],
                                [30, 20, 10], [5, 181, -3, 90], [7, 7, 3, 40, 60, 20, 170],
                                [*range(0, 100, 2), 3, *range(100, 180, 2)], [*range(0, 64), 500, *range(70, 170), 9]])
def test_rows_of_no_sequence_where_offsets_are_wrong(at):
    """They are zeros in a new output, wherever they lie, and stay as they are in a given one; rows of the good sequences are their own."""
    q, k, v = inputs([180], [180], 4, 2, 64, 3)
    good, fine = accepted(at, 180), torch.zeros(180, dtype=torch.bool, device="cuda")
    for out in (None, torch.full_like(q, 5)):
        leave_nan(q)
        got = ops.prompt_attention(q, k, v, i32(at), window=40, sinks=2, out=out)
        with pytest.raises(RuntimeError, match="offsets"):
            ops.check_device_errors()
        for a, b in good:
            fine[a:b] = True
            if b > a:
                check(got[a:b], q[a:b], k[a:b], v[a:b], [b - a], [b - a], 40, 2)
        assert (got[~fine] == (0 if out is None else 5)).all()


def test_rows_of_no_sequence_beside_parts():
    """The same where few queries with many keys are cut into parts."""
    q, k, v = inputs([300], [9000], 8, 2, 128, 4)
    leave_nan(q)
    got = ops.prompt_attention(q, k, v, i32([0, 100, 40, 220]), k_offsets=i32([0, 5000, 5000, 9000]))
    with pytest.raises(RuntimeError, match="offsets"):
        ops.check_device_errors()
    check(got[:100], q[:100], k[:5000], v[:5000], [100], [5000])
    assert (got[100:] == 0).all()


def test_keys_that_are_not_there():
    """Without any key, offsets of keys that claim one cannot be: NaN, and reported; a sequence of no keys beside it has zeros."""
    q = inputs([7], [7], 4, 2, 64, 1)[0]
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    got = ops.prompt_attention(q, none, none, i32([0, 2, 5, 7]), k_offsets=i32([0, 0, 1, 1]))
    with pytest.raises(RuntimeError, match="offsets"):
        ops.check_device_errors()
    assert (got[:2] == 0).all() and got[2:].isnan().all()  # the third one's keys begin behind the last row too
    assert (ops.prompt_attention(q, none, none, i32([0, 2, 5]), k_offsets=i32([0, 0, 0])) == 0).all()
    ops.check_device_errors()


def test_an_output_over_inputs():
    """Over the queries themselves, element for element, it is as good as any; anywhere else over what is read it is refused."""
    lengths = [90, 200, 10]
    for heads, kv_heads, keys in ((4, 2, None), (2, 2, [3000, 4000, 2000])):
        q, k, v = inputs(lengths, keys or lengths, heads, kv_heads, 128, 6)
        more = dict(window=30, sinks=2) if keys is None else dict(k_offsets=ends(keys))
        want = ops.prompt_attention(q, k, v, ends(lengths), **more)
        for _ in range(5):
            over = q.clone()
            assert ops.prompt_attention(over, k, v, ends(lengths), out=over, **more) is over
            assert torch.equal(over, want)
    q, k, v = inputs(lengths, lengths, 2, 2, 64, 7)
    buffer = torch.zeros(4 * 300 * 128, dtype=torch.bfloat16, device="cuda")
    at = lambda n: buffer[n * 128:(n + 300) * 128].view(300, 2, 64)  # noqa: E731
    for changes in (dict(k=at(0)), dict(v=at(0)), dict(k=at(299)), dict(v=at(299)), dict(q=at(1)), dict(q=at(299)),
                    dict(q=buffer[:300 * 256].view(300, 4, 64)[:, :2])):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.prompt_attention(**{**dict(q=q, k=k, v=v, offsets=ends(lengths)), **changes}, out=at(0))
    # side by side is not over one another
    ops.prompt_attention(at(0), at(300), at(600), ends(lengths), out=at(900))
    ops.check_device_errors()


@pytest.mark.parametrize("keys", [300, 5000])
def test_a_scale_that_is_nan(keys):
    q, k, v = inputs([300], [keys], 4, 2, 128, 8)
    assert ops.prompt_attention(q, k, v, ends([300]), scale=math.nan, k_offsets=ends([keys])).isnan().all()


@pytest.mark.parametrize("dim,group", [(128, 4), (64, 1)])
@pytest.mark.parametrize("keys", [200, 5000])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_the_row_that_sees_a_key_that_is_not_finite(dim, group, keys, value):
    """A score of NaN or +inf makes its head's row NaN, a score of -inf is a key that does not count."""
    q, k, v = inputs([200], [keys], 2 * group, 2, dim, 9)
    k[keys - 1, 1, 3] = value
    got = ops.prompt_attention(q, k, v, ends([200]), k_offsets=ends([keys]))
    want, size, _ = definition64(q, k, v, [200], [keys], 0, 0, dim ** -0.5)
    k[keys - 1] = 0
    reach = definition64(q, k, v, [200], [keys], 0, 0, dim ** -0.5)[2]
    spoilt = torch.zeros(2 * group, dtype=torch.bool, device="cuda")
    spoilt[group:] = True if math.isnan(value) else q[199, group:, 3] * value > 0
    assert torch.equal(got[199].isnan().all(-1), spoilt) and torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    assert ((got.double() - want).abs() <= bound(want, size, reach, dim, keys))[fine].all()
    ops.check_device_errors()
