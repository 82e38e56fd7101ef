"""A server's steps: places and pages planned on the device, append, attention with a window, rules on the logits, one behind the other and in the decoder."""
import pytest
import torch

from sharq_b200 import ops
from tests import paged_util as P
from tests.test_decode_gpu import small, tokens
from tests.test_logit_rules_gpu import check as check_logits, rules64
from tests.test_prompt_attention_gpu import bound as prompt_bound, definition64 as prompt64
from tests.test_windowed_attention_gpu import definition64 as token64

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page,window,sinks", [(16, 30, 4), (24, 8, 0), (64, 1000, 3)])
def test_plan_append_attention_rules(page, window, sinks):
    """Prompts come and go while other sequences decode; every operator against its definition on the inputs that it had."""
    seqs, heads, kv, dim, most = 5, 8, 2, 128, 12
    g = torch.Generator(device="cuda").manual_seed(page)
    pages = seqs * most
    table, lengths, stack, free = i32([[-1] * most] * seqs), i32([0] * seqs), torch.arange(pages, device="cuda", dtype=torch.int32), i32([pages])
    k_cache, v_cache, *_ = P.make_cache(pages, kv, page, dim, False, 2)
    cos, sin = P.rope_tables(most * page, dim)
    history, held = torch.full((seqs, 64), -1, dtype=torch.int32, device="cuda"), i32([0] * seqs)

    def step(counts, released):
        rows = sum(counts) + 3
        offsets, positions, which = ops.plan_paged_step(table, lengths, i32(counts), stack, free, page, rows, released=torch.tensor(released, device="cuda"))
        qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g, device="cuda").to(torch.bfloat16)
        q, k = ops.rope_append_paged(qkv, heads, kv, dim, cos, sin, positions, table, k_cache, v_cache, sequences=which, return_k=True)
        v = qkv[:, (heads + kv) * dim:].view(rows, kv, dim)
        return offsets, positions, which, q, k, v

    # prompts: the keys are those of the step
    for counts, released in (([7, 0, 90, 33, 1], [False] * 5), ([0, 41, 0, 0, 60], [False, False, True, False, True])):
        offsets, positions, which, q, k, v = step(counts, released)
        got = ops.prompt_attention(q, k, v, offsets, window=window, sinks=sinks)
        n = sum(counts)
        want, size, reach = prompt64(q[:n], k, v, counts, counts, window, sinks, dim ** -0.5)
        assert ((got[:n].double() - want).abs() <= prompt_bound(want, size, reach, dim, 90)).all() and (got[n:] == 0).all()
        at = positions[:n].long()
        kept = table[which[:n].long(), at // page].long(), slice(None), at % page
        assert torch.equal(k_cache[kept], k[:n]) and torch.equal(v_cache[kept], v[:n])
    assert lengths.tolist() == [7, 41, 0, 33, 60]
    assert int(free) == pages - sum(-(-n // page) for n in lengths.tolist())
    # single tokens, in rows of their sequences
    for i in range(20):
        _, positions, which, q, _, _ = step([1] * seqs, [False] * seqs)
        got = ops.paged_attention(q[:seqs], k_cache, v_cache, table, lengths, window=window, sinks=sinks)
        want, size, reach = token64(q[:seqs], k_cache.double(), v_cache.double(), table, lengths.tolist(), window, sinks, dim ** -0.5)
        assert ((got.double() - want).abs() <= P.attention_bound(want, size, reach, dim, window + sinks, False)).all()
        logits = got.float().flatten(1) * 3
        rules = dict(tokens=history, lengths=held, presence=torch.full((seqs,), 0.5, device="cuda"), repetition=torch.full((seqs,), 1.2, device="cuda"))
        out = ops.adjust_logits(logits, **rules)
        check_logits(logits, out, rules64(logits, **rules))
        history[:, i] = out.argmax(-1).int()
        held += 1
    assert lengths.tolist() == [27, 61, 20, 53, 80] and positions[:seqs].tolist() == [26, 60, 19, 52, 79] and which[:seqs].tolist() == [0, 1, 2, 3, 4]
    assert len(set(table[s, j].item() for s in range(seqs) for j in range(-(-int(lengths[s]) // page)))) == pages - int(free)
    ops.check_device_errors()


@pytest.mark.parametrize("kw", [dict(window=20, sinks=4), dict(window=33, sinks=0, head_dim=64, heads=4, kv_heads=4), dict(window=1, sinks=1), dict(window=500, sinks=2)])
def test_a_model_with_a_window(kw):
    """The kernels against the composition of library operators with a mask, in unquantised layers; decode steps against the prompt with those tokens.
    The bound is that of decode steps without a window: some twenty roundings of half a step of bf16 in sequence over the two layers, at most 8 %."""
    from sharq_b200.decoder import SharqDecoder

    cfg = small(**kw)
    fused, plain = (SharqDecoder(cfg, torch.device("cuda"), mode="BF16", fused_glue=f, seed=3) for f in (True, False))
    ids = tokens(cfg, 3, 130)
    want = plain.prefill(ids)
    assert (fused.prefill(ids) - want).norm() <= 0.08 * want.norm()
    if cfg.window < 130:
        cfg_all = small(**{**kw, "window": 0, "sinks": 0})
        other = SharqDecoder(cfg_all, torch.device("cuda"), mode="BF16", fused_glue=False, seed=3).prefill(ids)
        assert (other - want).norm() > 0.08 * want.norm()  # the window matters
    cache = fused.new_cache(3, 140, page_size=16)
    fused.prefill(ids[:, :126], cache=cache)
    for i in range(126, 130):
        got = fused.decode(ids[:, i], cache)
    assert (got - want).norm() <= 0.08 * want.norm()
    quantised = SharqDecoder(cfg, torch.device("cuda"), seed=3)
    cache = quantised.new_cache(3, 140, page_size=16)
    assert quantised.prefill(ids, cache=cache).isfinite().all() and quantised.decode(ids[:, 0], cache, weight_only=True).isfinite().all()
    ops.check_device_errors()


@pytest.mark.parametrize("window", [0, 20])
def test_pages_from_the_device_are_those_from_the_host(window):
    from sharq_b200.decoder import SharqDecoder

    cfg = small(window=window, sinks=4)
    model = SharqDecoder(cfg, torch.device("cuda"), mode="BF16", seed=3)
    ids = tokens(cfg, 4, 60)
    host, device = (model.new_cache(4, 80, page_size=16, pages=18, on_device=d) for d in (False, True))

    def same():
        n = host.lengths
        assert device.device_lengths.tolist() == host.device_lengths.tolist() == n
        for i, held in enumerate(host._held):
            assert device.table[i, :len(held)].tolist() == held
        assert device.free_pages[:int(device.free_count)].tolist() == host._free

    for cache in (host, device):
        a = model.prefill(ids[[2, 0], :45], cache=cache, sequences=[2, 0])
        b = model.prefill(ids[[1, 3], :30], cache=cache, sequences=[1, 3])
        cache.first = a, b
    same()
    for x, y in zip(host.first, device.first):
        assert torch.equal(x, y)
    for i in range(45, 52):
        got = [model.decode(ids[:, i], cache) for cache in (host, device)]
        assert (got[0] - got[1]).norm() <= 0.08 * got[0].norm()
        got = [model.decode(ids[[3, 1], i], cache, sequences=[3, 1]) for cache in (host, device)]
        assert (got[0] - got[1]).norm() <= 0.08 * got[0].norm()
        same()
    for cache in (host, device):
        cache.free(2)
    same()
    # a prompt in the place of a sequence that goes on
    host.free(1)
    assert torch.equal(*(model.prefill(ids[1:2], cache=cache, sequences=[1]) for cache in (host, device)))
    same()
    # pages that do not suffice: the host refuses the step, the device leaves out the sequences that they do not reach
    model.prefill(ids[2:3], cache=device, sequences=[2])
    before = device.device_lengths.tolist()
    while int(device.free_count) > 0:
        model.decode(ids[:, 0], device)
    full = device.device_lengths.tolist()
    for _ in range(16):
        logits = model.decode(ids[:, 0], device)
    assert all(n - (n - 1) // 16 * 16 == 16 or n == 80 for n in device.device_lengths.tolist()) and min(b - a for a, b in zip(before, full)) >= 1
    assert logits.isfinite().all()
    ops._ERROR_FLAGS[0].zero_()  # one of them may have reached 80


def test_host_and_device_do_not_mix():
    from sharq_b200.decoder import SharqDecoder

    cfg = small()
    model = SharqDecoder(cfg, torch.device("cuda"), seed=3)
    host, device = (model.new_cache(2, 64, page_size=16, on_device=d) for d in (False, True))
    counts = torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="host"):
        host.plan(counts, 2)
    for call in (lambda: device.reserve([1, 1]), lambda: device.advance([1, 1]), lambda: device.prompt_step(3)):
        with pytest.raises(RuntimeError, match="device"):
            call()
    ids = tokens(cfg, 3, 70)
    for bad in (ids, ids[:2]):
        with pytest.raises(ValueError, match="prompt"):
            model.prefill(bad, cache=device)
    model.prefill(ids[:2, :64], cache=device)
    model.decode(ids[:2, 0], device)  # beyond max_tokens
    assert device.device_lengths.tolist() == [64, 64]
    with pytest.raises(RuntimeError, match="plan_paged_step"):
        ops.check_device_errors()


def test_a_captured_step_grows_its_sequences():
    """Pages, attention, rules and the choice of a token in one graph, replayed from token to token as the eager steps go."""
    from sharq_b200.decoder import SharqDecoder
    from sharq_b200.logit_rules import LogitRules

    cfg = small(window=25, sinks=3)
    model = SharqDecoder(cfg, torch.device("cuda"), seed=3)
    ids = tokens(cfg, 2, 20)

    def begin():
        cache = model.new_cache(2, 200, page_size=16, on_device=True)
        history = torch.zeros(2, 200, dtype=torch.int64, device="cuda")
        history[:, :20] = ids
        rules = LogitRules(tokens=history, lengths=i32([20, 20]), prompt_lengths=i32([20, 20]), repetition=torch.full((2,), 1.3, device="cuda"),
                           frequency=torch.full((2,), 0.2, device="cuda"), bias=(i32([0, 1, 1]), i32([7]), torch.ones(1, device="cuda")),
                           mask=torch.full((2, -(-cfg.vocab // 32)), 0x55555555, dtype=torch.int32, device="cuda"))
        return cache, rules, model.prefill(ids, cache=cache, rules=rules).argmax(-1)

    def step(token, cache, rules):
        rules.append_(token)
        logits = model.decode(token, cache, rules=rules)
        token.copy_(logits.argmax(-1))
        return logits

    cache, rules, token = begin()
    assert (token % 2 == 0).all()
    eager = []
    for _ in range(60):
        eager.append((step(token, cache, rules).clone(), token.clone()))
    cache, rules, token = begin()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = begin()
        step(warm[2], warm[0], warm[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = step(token, cache, rules)
    for want, chosen in eager:
        graph.replay()
        assert torch.equal(logits, want) and torch.equal(token, chosen)
    assert cache.device_lengths.tolist() == [80, 80] and rules.lengths.tolist() == [80, 80]
    # what the rules do to logits is what the operator does
    plain = model.decode(token, cache)
    cache2, rules2, _ = begin()
    assert (model.prefill(ids, cache=cache2)[:, 1::2].isfinite()).all() and plain.isfinite().all()
    first = model.prefill(ids)
    assert torch.equal(model.prefill(ids, rules=rules2), ops.adjust_logits(first, rules2.tokens, rules2.lengths, rules2.prompt_lengths, rules2.repetition,
                                                                           rules2.presence, rules2.frequency, rules2.bias, rules2.mask))
    ops.check_device_errors()
