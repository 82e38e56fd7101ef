"""Caches that hand their pages out on the device, where the pages do not suffice or an argument is refused."""
import pytest
import torch

from sharq_b200 import ops
from tests.test_decode_gpu import small, tokens

pytestmark = pytest.mark.gpu


def model_of(**kw):
    from sharq_b200.decoder import SharqDecoder

    cfg = small(**kw)
    return SharqDecoder(cfg, torch.device("cuda"), mode="BF16", seed=3), cfg


@pytest.mark.parametrize("window", [0, 20])
def test_a_prompt_without_pages_is_reported_and_nothing_follows_it(window):
    model, cfg = model_of(window=window, sinks=4 if window else 0)
    ids = tokens(cfg, 3, 33)
    cache = model.new_cache(3, 64, page_size=16, pages=5, on_device=True)
    logits = model.prefill(ids, cache=cache)  # three pages each: the first one's, and no others
    with pytest.raises(RuntimeError, match="pages"):
        ops.check_device_errors()
    assert logits[0].isfinite().all() and logits[1:].isnan().all()
    for _ in range(2):  # two pages are free, but a token without its prompt does not take one
        model.decode(ids[:, 0], cache)
        with pytest.raises(RuntimeError, match="plan_paged_step"):
            ops.check_device_errors()
    assert cache.device_lengths.tolist() == [35, -1, -1] and int(cache.free_count) == 2
    # where there is room the prompt takes its place after all, and steps go on from it
    cache.free(0)
    other = model.new_cache(3, 64, page_size=16, on_device=True)
    for c in (cache, other):
        c.first = model.prefill(ids[1:2], cache=c, sequences=[1])
        c.second = model.decode(ids[[1], 4], c, sequences=[1])
    assert torch.equal(cache.first, other.first) and (cache.second - other.second).norm() <= 0.08 * other.second.norm()
    cache.free(2)
    assert cache.device_lengths.tolist() == [0, 34, 0] and int(cache.free_count) == 2
    model.decode(ids[[2], 0], cache, sequences=[2])  # a sequence that is empty and waits for nothing begins with a token
    assert cache.device_lengths.tolist() == [0, 34, 1]
    ops.check_device_errors()


def test_tokens_without_pages_are_reported():
    model, cfg = model_of()
    ids = tokens(cfg, 2, 20)
    cache = model.new_cache(2, 64, page_size=16, pages=3, on_device=True)
    model.prefill(ids[:, :15], cache=cache)
    model.decode(ids[:, 15], cache)
    ops.check_device_errors()
    assert model.decode(ids[:, 16], cache).isfinite().all()
    with pytest.raises(RuntimeError, match="pages"):
        ops.check_device_errors()
    assert cache.device_lengths.tolist() == [17, 16]
    cache.free(0)
    model.decode(ids[[1], 16], cache, sequences=[1])  # the same token again, now that there is a page
    assert cache.device_lengths.tolist() == [0, 17]
    ops.check_device_errors()


def test_plans_report_a_shortage_where_they_are_asked_to():
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for strict in (False, True):
        for counts, free, short in (([1, 1, 1], 2, True), ([0, 1, 0], 0, True), ([1, 0, 1], 2, False), ([0, 0, 0], 0, False)):
            lengths, left = dev([16, 16, 32]), dev([free])
            got = ops.plan_paged_step(torch.zeros(3, 4, dtype=torch.int32, device="cuda"), lengths, dev(counts), dev(list(range(9))), left, 16, 3, strict=strict)
            if short and strict:
                with pytest.raises(RuntimeError, match="pages"):
                    ops.check_device_errors()
            ops.check_device_errors()
            taken = [n for n in (torch.tensor(counts).cumsum(0)).tolist()]
            assert lengths.tolist() == [n + (c if t <= free else 0) for n, c, t in zip([16, 16, 32], counts, taken)]
            assert len(got) == 3


def test_rules_of_other_rows_are_refused_before_anything_changes():
    from sharq_b200.logit_rules import LogitRules

    model, cfg = model_of()
    ids = tokens(cfg, 2, 9)
    rules = LogitRules(tokens=ids.clone(), lengths=torch.full((2,), 9, dtype=torch.int32, device="cuda"))
    for on_device in (False, True):
        cache = model.new_cache(2, 64, page_size=16, on_device=on_device)
        with pytest.raises((ValueError, RuntimeError)):
            model.prefill(ids[:1], cache=cache, sequences=[1], rules=rules)
        assert cache.device_lengths.tolist() == [0, 0]
        model.prefill(ids, cache=cache, rules=rules)
        with pytest.raises((ValueError, RuntimeError)):
            model.decode(ids[1:, 0], cache, sequences=[1], rules=rules)
        assert cache.device_lengths.tolist() == [9, 9]
        model.decode(ids[:, 0], cache, rules=rules)
        assert cache.device_lengths.tolist() == [10, 10]
    ops.check_device_errors()


def test_steps_of_a_full_cache_report_the_plan_and_nothing_else():
    """Steps go on, captured ones too, with some sequences left out; neither the append nor the attention has anything to say about them."""
    model, cfg = model_of(window=20, sinks=3)
    ids = tokens(cfg, 4, 30)
    cache = model.new_cache(4, 48, page_size=16, pages=9, on_device=True)
    model.prefill(ids[:, :30], cache=cache)
    ops.check_device_errors()
    token = ids[:, 0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.decode(token, cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.decode(token, cache)
    codes = []
    for _ in range(20):
        graph.replay()
        codes.append(int(ops._ERROR_FLAGS[0]))
        ops._ERROR_FLAGS[0].zero_()
        assert logits.isfinite().all()
    # 31 tokens each; all grow to 32, then the first one alone, which gets the last page, up to max_tokens
    assert cache.device_lengths.tolist() == [48, 32, 32, 32] and int(cache.free_count) == 0
    # no error, then pages that do not suffice, and from 48 on either that or a length that cannot be, whichever comes first
    assert codes[:17] == [0] + [0x409] * 16 and set(codes[17:]) <= {0x405, 0x409}
    ops.check_device_errors()
