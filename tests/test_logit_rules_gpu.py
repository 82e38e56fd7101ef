"""Penalties, biases and masks on logits (ops.adjust_logits) against their formulas in 64 bits."""
import math

import pytest
import torch

from sharq_b200 import ops

pytestmark = pytest.mark.gpu


def rules64(logits, tokens=None, lengths=None, prompt_lengths=None, repetition=None, presence=None, frequency=None, bias=None, mask=None):
    """Row by row, token by token, in 64 bits."""
    out = logits.double().clone()
    rows, vocab = out.shape
    lengths, prompt_lengths = (x if x is None else x.tolist() for x in (lengths, prompt_lengths))
    for i in range(rows):
        if tokens is not None:
            n = min(max(lengths[i], 0), tokens.shape[1])
            history = tokens[i, :n].long()
            made = history[max(0, prompt_lengths[i]):] if prompt_lengths is not None else history
            there = lambda x: x[(x >= 0) & (x < vocab)]  # noqa: E731
            seen, counts = there(history).unique(), torch.bincount(there(made), minlength=vocab)
            if repetition is not None:
                x, r = out[i, seen], repetition[i].double()
                out[i, seen] = torch.where(x > 0, x / r, x * r)
            hit = counts.nonzero()[:, 0]
            if frequency is not None:
                out[i, hit] -= frequency[i].double() * counts[hit]
            if presence is not None:
                out[i, hit] -= presence[i].double()
        if bias is not None:
            a, b = int(bias[0][i]), int(bias[0][i + 1])
            if 0 <= a <= b <= bias[1].numel():
                row = out[i].tolist()
                for token, value in zip(bias[1][a:b].tolist(), bias[2][a:b].double().tolist()):
                    if 0 <= token < vocab:
                        row[token] += value
                out[i] = torch.tensor(row, dtype=torch.float64)
        if mask is not None:
            token = torch.arange(vocab, device=out.device)
            out[i, (mask[i].long()[token // 32] >> (token % 32)) & 1 == 0] = -math.inf
    return out


def check(logits, got, want):
    """One rounding from 64 bits: half a step of the type, and half a step again for a product that 64 bits have not decided."""
    assert got.dtype == logits.dtype and got.shape == logits.shape
    got = got.double()
    bound = torch.finfo(logits.dtype).eps / 2 * (1 + 1e-6) * want.abs() + torch.finfo(torch.float32).tiny
    assert ((got == want) | ((got - want).abs() <= bound) | (got.isnan() & want.isnan())).all()


def case(rows, vocab, width, seed, dtype=torch.float32, ids=torch.int32, biases=0, mask=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    logits = (3 * torch.randn(rows, vocab, generator=g, device="cuda")).to(dtype)
    tokens = (rand(rows, width) ** 3 * vocab).long().clamp(max=vocab - 1).to(ids)
    lengths = (rand(rows) * (width + 1)).int().clamp(max=width)
    rules = dict(tokens=tokens, lengths=lengths, prompt_lengths=(lengths * rand(rows)).int(), repetition=0.8 + rand(rows), presence=rand(rows) - 0.3,
                 frequency=0.3 * rand(rows))
    if biases:
        offsets = torch.cat((torch.zeros(1, device="cuda"), (rand(rows) * 2 * biases).int().cumsum(0))).int()
        n = int(offsets[-1])
        rules["bias"] = (offsets, (rand(n) * vocab).int().clamp(max=vocab - 1), 5 * torch.randn(n, generator=g, device="cuda"))
    if mask:
        rules["mask"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g, device="cuda").int()
    return logits, rules


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,vocab,width,biases", [(1, 1, 1, 0), (1, 33, 5, 3), (3, 128256, 700, 9), (2, 4099, 0, 4), (65, 1000, 77, 0), (7, 32000, 3001, 500),
                                                     (300, 517, 40, 20), (1, 152064, 20000, 4000)])
def test_rows_against_the_formulas(dtype, ids, rows, vocab, width, biases):
    logits, rules = case(rows, vocab, width, rows + vocab, dtype, ids, biases)
    kept = logits.clone()
    check(logits, ops.adjust_logits(logits, **rules), rules64(logits, **rules))
    assert torch.equal(logits, kept)
    assert ops.adjust_logits(logits, out=logits, **rules) is logits
    check(kept, logits, rules64(kept, **rules))
    ops.check_device_errors()


@pytest.mark.parametrize("left", ["tokens", "prompt_lengths", "repetition", "presence", "frequency", "bias", "mask"])
def test_each_rule_alone_and_each_left_out(left):
    logits, rules = case(5, 3001, 200, 9, biases=7)
    history = ("tokens", "lengths", "prompt_lengths", "repetition", "presence", "frequency")
    out = {left} if left != "tokens" else set(history)
    some = {k: v for k, v in rules.items() if k not in out}
    check(logits, ops.adjust_logits(logits, **some), rules64(logits, **some))
    some = {k: v for k, v in rules.items() if k in out or (k in ("tokens", "lengths") and left in history)}
    check(logits, ops.adjust_logits(logits, **some), rules64(logits, **some))
    assert torch.equal(ops.adjust_logits(logits), logits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_unaligned_rows(dtype):
    logits, rules = case(6, 1001, 90, 3, dtype, biases=5)
    wide = torch.full((6, 1013), 7.0, dtype=dtype, device="cuda")
    wide[:, 5:1006] = logits
    rules["tokens"] = torch.cat((rules["tokens"], rules["tokens"]), 1)[:, 90:]
    rules["mask"] = torch.cat((rules["mask"], rules["mask"]), 1)[:, :32]
    want = rules64(logits, **rules)
    check(logits, ops.adjust_logits(wide[:, 5:1006], **rules), want)
    to = torch.full((6, 1016), 7.0, dtype=dtype, device="cuda")
    check(logits, ops.adjust_logits(logits, out=to[:, 8:1009], **rules), want)
    assert (to[:, :8] == 7).all() and (to[:, 1009:] == 7).all()
    ops.adjust_logits(wide[:, 5:1006], out=wide[:, 5:1006], **rules)
    check(logits, wide[:, 5:1006], want)
    assert (wide[:, :5] == 7).all() and (wide[:, 1006:] == 7).all()
    # one history and one mask for all rows
    for name in ("tokens", "mask"):
        rules[name] = rules[name][:1].expand(6, -1)
    check(logits, ops.adjust_logits(logits, **rules), rules64(logits, **rules))


def test_the_same_token_again_and_again():
    """A token many times in the history, and with many biases, which add up in any number of calls to the same bits."""
    logits, rules = case(4, 700, 5000, 5, biases=0)
    rules["tokens"][:, ::2] = 699
    ids = torch.tensor([3, 699, 3, 3, 699, 5] * 400, device="cuda", dtype=torch.int32)
    values = torch.randn(2400, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 10.0 ** (torch.arange(2400, device="cuda") % 7 - 3)
    rules["bias"] = (torch.tensor([0, 600, 600, 1800, 2400], device="cuda", dtype=torch.int32), ids, values)
    got = ops.adjust_logits(logits, **rules)
    # the sums of a few hundred values of up to 10^4: in 64 bits their order says less than a step of the result, unless it nearly cancels
    want = rules64(logits, **rules)
    assert ((got.double() - want).abs() <= 2.0 ** -24 * (1 + 1e-6) * want.abs() + 1e-9).logical_or(got.double() == want).all()
    for _ in range(5):
        assert torch.equal(got, ops.adjust_logits(logits, **rules))


def test_values_that_are_not_finite():
    logits, rules = case(3, 400, 300, 6, biases=6)
    logits[:, ::7], logits[:, 1::7], logits[:, 2::7] = math.inf, -math.inf, math.nan
    got = ops.adjust_logits(logits, **rules)
    check(logits, got, rules64(logits, **rules))
    token = torch.arange(400, device="cuda")
    masked = (rules["mask"].long()[:, token // 32] >> (token % 32)) & 1 == 0
    assert (got[masked] == -math.inf).all()
    rules["mask"].zero_()
    assert (ops.adjust_logits(logits, **rules) == -math.inf).all()


def test_what_is_out_of_range_is_passed_over():
    logits, rules = case(3, 1000, 50, 7, biases=4)

    def reported(**changes):
        some = {**rules, **changes}
        check(logits, ops.adjust_logits(logits, **some), rules64(logits, **some))
        with pytest.raises(RuntimeError, match="adjust_logits"):
            ops.check_device_errors()

    tokens = rules["tokens"].clone()
    tokens[:, ::3] = -1
    tokens[:, 1::3] = -2 ** 31
    check(logits, ops.adjust_logits(logits, **{**rules, "tokens": tokens}), rules64(logits, **{**rules, "tokens": tokens}))
    ops.check_device_errors()  # padding
    full = torch.tensor([50, 50, 50], dtype=torch.int32, device="cuda")
    for token in (1000, 2 ** 31 - 1):
        tokens[1, 0] = token
        reported(tokens=tokens, lengths=full)
    reported(tokens=tokens.long() << 24, lengths=full)
    reported(lengths=torch.tensor([51, 3, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    reported(lengths=torch.tensor([5, -1, 50], dtype=torch.int32, device="cuda"))
    offsets, ids, values = rules["bias"]
    n = ids.numel()
    for bad in ([0, 3, 2, n], [0, 3, 5, n + 1], [-1, 3, 5, n]):
        reported(bias=(torch.tensor(bad, dtype=torch.int32, device="cuda"), ids, values))
    ids = ids.clone()
    ids[0], ids[1] = 1000, -1
    offsets = torch.tensor([0, 2, 2, n], dtype=torch.int32, device="cuda")
    reported(bias=(offsets, ids, values))
    check(logits, ops.adjust_logits(logits, **{**rules, "prompt_lengths": torch.tensor([-5, 99, 0], dtype=torch.int32, device="cuda")}),
          rules64(logits, **{**rules, "prompt_lengths": torch.tensor([-5, 99, 0], dtype=torch.int32, device="cuda")}))
    ops.check_device_errors()


def test_captured_and_on_another_stream():
    logits, rules = case(4, 32000, 500, 8, biases=9)
    want = rules64(logits, **rules)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.adjust_logits(logits, **rules)
    torch.cuda.current_stream().wait_stream(side)
    check(logits, got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.adjust_logits(logits, **rules)
    rules["lengths"][0] = 0
    logits[1] *= -1
    graph.replay()
    check(logits, got, rules64(logits, **rules))


def test_no_rows_and_refusals():
    logits, rules = case(3, 100, 20, 1, biases=3)
    none = torch.zeros(0, 100, device="cuda")
    assert ops.adjust_logits(none).shape == (0, 100)
    dev = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    offsets, ids, values = rules["bias"]
    overlap = torch.zeros(3 * 100 + 1, device="cuda")
    for name, value in [("tokens", None), ("lengths", None), ("tokens", dev(2, 20)), ("tokens", dev(3, 20, t=torch.int16)), ("tokens", dev(20, 3).T), ("tokens", dev(3, 20).cpu()),
                        ("lengths", dev(4)), ("lengths", dev(3, t=torch.int64)), ("prompt_lengths", dev(2)), ("repetition", dev(3)),
                        ("presence", dev(2, t=torch.float32)), ("frequency", dev(3, t=torch.float64)), ("bias", (offsets, ids)),
                        ("bias", (offsets[:-1].contiguous(), ids, values)), ("bias", (offsets, ids.long(), values)), ("bias", (offsets, ids, values[:-1])),
                        ("mask", dev(3, 3)), ("mask", dev(3, 5)), ("mask", dev(3, 4, t=torch.int64)), ("mask", dev(2, 4)), ("out", dev(3, 100)),
                        ("out", dev(3, 101, t=torch.float32)), ("out", logits.cpu())]:
        with pytest.raises((RuntimeError, TypeError)):
            ops.adjust_logits(logits, **{**rules, name: value})
    with pytest.raises(RuntimeError, match="overlap"):
        ops.adjust_logits(overlap[:300].view(3, 100), out=overlap[1:].view(3, 100))
    with pytest.raises(RuntimeError, match="overlap"):
        ops.adjust_logits(logits[:1].expand(3, 100), **rules)
    for bad in (logits.half(), logits[0], logits.T, logits.cpu(), logits[:, :0]):
        with pytest.raises(RuntimeError):
            ops.adjust_logits(bad)
    with pytest.raises(RuntimeError, match="need tokens"):
        ops.adjust_logits(logits, presence=dev(3, t=torch.float32))
