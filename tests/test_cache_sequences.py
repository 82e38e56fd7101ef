"""Sequences of one paged cache that begin, go on and end apart from one another."""
import pytest
import torch

from sharq_b200.decoder import rope_tables
from sharq_b200.kv_cache import PagedKVCache


def make(**kw):
    cos, sin = rope_tables(40, 64, 1e4, torch.device("cpu"))
    return PagedKVCache(1, 2, 64, 3, 40, cos, sin, 8, **kw)


def test_a_step_of_some_sequences():
    cache = make()
    assert cache.chosen(None) == [0, 1, 2] and cache.chosen((2, 0)) == [2, 0] and cache.counts([2, 0], 5) == [5, 0, 5]
    cache.reserve(cache.counts([2, 0], 9))
    cache.advance(cache.counts([2, 0], 9))
    assert cache.lengths == cache.device_lengths.tolist() == [9, 0, 9]
    cache.reserve([2, 4, 0])
    positions, sequences = cache.prompt_step(2, [1, 0])
    assert positions.tolist() == [0, 1, 9, 10] and sequences.tolist() == [1, 1, 0, 0]
    assert positions.dtype == sequences.dtype == torch.int32
    rows = torch.tensor([2, 1])
    assert cache.held_table().shape == (3, 2) and torch.equal(cache.held_table(rows), cache.table[[2, 1], :2])
    layer = cache.layer(0, positions, None, None, cache.held_table(rows))
    assert torch.equal(layer.table, cache.table[[2, 1], :2])
    assert torch.equal(cache.layer(0, positions, None, None).table, cache.table[:, :2])
    strange = cache.held_table(torch.tensor([1, 3, -1, 2 ** 40]))  # of no sequence: no pages
    assert torch.equal(strange[0], cache.table[1, :2]) and bool((strange[1:] == -1).all()) and strange.dtype == torch.int32


@pytest.mark.parametrize("sequences", [[], [3], [-1], [0, 0], [0, 1, 2, 0]])
def test_lists_that_are_refused(sequences):
    with pytest.raises(ValueError, match="different numbers below 3"):
        make().chosen(sequences)


def small(**kw):
    from sharq_b200.decoder import DecoderConfig

    return DecoderConfig(**{**dict(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=128, ffn=1024, vocab=2000), **kw})


@pytest.mark.gpu
@pytest.mark.parametrize("reference", [False, True])
def test_another_prompt_in_a_freed_place(reference):
    """Three sequences; the second ends, a new prompt takes its place while the others go on.  Each sequence then gives what it gives in a
    cache of its own.  The linears' products of a row do not depend on the other rows (weight_only; with reference=True their sums may), the
    attention's order of sums may: some 25 roundings of 2^-8 in sequence over the two layers differ at most, 10 %."""
    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg, dev = small(), torch.device("cuda")
    model = SharqDecoder(cfg, dev, keep_reference=reference, seed=3)
    ids = torch.randint(0, cfg.vocab, (4, 60), generator=torch.Generator().manual_seed(1)).cuda()
    kw = dict(reference=True) if reference else dict(weight_only=True)

    def alone(row, prompt, steps):
        cache = model.new_cache(1, 64, page_size=16)
        model.prefill(ids[row:row + 1, :prompt], reference=reference, cache=cache)
        out = [model.decode(ids[row:row + 1, prompt + i], cache, **kw)[0] for i in range(steps)]
        return out, cache

    prompts, want = {0: 20, 1: 33, 2: 5, 3: 17}, {}
    for row, steps in ((0, 8), (1, 3), (2, 4), (3, 5)):
        want[row], _ = alone(row, prompts[row], steps)

    cache = model.new_cache(3, 64, page_size=16, pages=8)  # the new prompt needs pages that were given back
    for row in range(3):
        model.prefill(ids[row:row + 1, :prompts[row]], reference=reference, cache=cache, sequences=[row])
    assert cache.lengths == [20, 33, 5]
    at, got = dict(prompts), {row: [] for row in range(4)}

    def step(rows):
        """rows: the row of ids that goes on in each listed sequence."""
        token = torch.stack([ids[row, at[row]] for row in rows.values()])
        logits = model.decode(token, cache, sequences=list(rows), **kw)
        for row, out in zip(rows.values(), logits):
            got[row].append(out.clone())
            at[row] += 1

    for _ in range(3):
        step({0: 0, 1: 1})
    cache.free(1)
    with pytest.raises(ValueError, match="one empty sequence"):
        model.prefill(ids[3:4, :17], cache=cache, sequences=[0])
    held = [cache._held[i][:-(-n // 16)] for i, n in ((0, cache.lengths[0]), (2, cache.lengths[2]))]
    before = [cache.k[:, pages].view(torch.int16) for pages in held]  # as bits: slots behind a sequence hold anything
    model.prefill(ids[3:4, :17], reference=reference, cache=cache, sequences=[1])
    assert all(torch.equal(cache.k[:, pages].view(torch.int16), was) for pages, was in zip(held, before))
    for _ in range(4):
        step({2: 2, 0: 0, 1: 3})  # in any order
    step({1: 3, 0: 0})
    ops.check_device_errors()
    assert cache.lengths == cache.device_lengths.tolist() == [28, 22, 9]
    for row in range(4):
        assert len(got[row]) == len(want[row])
        for a, b in zip(got[row], want[row]):
            assert (a - b).norm() <= 0.1 * b.norm(), row


@pytest.mark.gpu
def test_a_captured_step_of_some_sequences():
    """A graph reads which sequences it is for, as it reads their lengths, when it is replayed."""
    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg = small()
    model = SharqDecoder(cfg, torch.device("cuda"), seed=3)
    ids = torch.randint(0, cfg.vocab, (3, 30), generator=torch.Generator().manual_seed(1)).cuda()
    caches = [model.new_cache(3, 64, page_size=16) for _ in range(2)]
    for cache in caches:
        for row, n in enumerate((20, 3, 11)):
            model.prefill(ids[row:row + 1, :n], cache=cache, sequences=[row])
    cache = caches[0]
    eager = [model.decode(ids[rows, 20 + i], cache, weight_only=True, sequences=rows).clone() for i, rows in enumerate(([2, 0], [0, 1], [1, 2]))]
    cache = caches[1]
    cache.reserve([2, 2, 2])
    rows = torch.tensor([2, 0]).cuda()
    token, positions, lengths = ids[rows, 20], cache.device_lengths[rows], cache.device_lengths[rows] + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.decode_step(token, cache, positions, lengths, weight_only=True, rows=rows)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.decode_step(token, cache, positions, lengths, weight_only=True, rows=rows)
    for i, which in enumerate(([2, 0], [0, 1], [1, 2])):
        rows.copy_(torch.tensor(which))
        token.copy_(ids[which, 20 + i])
        positions.copy_(cache.device_lengths[which])
        lengths.copy_(cache.device_lengths[which] + 1)
        graph.replay()
        cache.advance(cache.counts(which, 1))
        assert torch.equal(logits, eager[i])
    ops.check_device_errors()


@pytest.mark.gpu
def test_refusals_of_some_sequences():
    from sharq_b200.decoder import SharqDecoder

    cfg = small()
    model = SharqDecoder(cfg, torch.device("cuda"), seed=3)
    ids = torch.randint(0, cfg.vocab, (3, 5), generator=torch.Generator().manual_seed(1)).cuda()
    cache = model.new_cache(3, 8, page_size=4)
    with pytest.raises(ValueError, match="of a cache"):
        model.prefill(ids, sequences=[0, 1, 2])
    with pytest.raises(ValueError, match="one empty sequence"):
        model.prefill(ids, cache=cache, sequences=[0, 1])
    with pytest.raises(ValueError, match="different numbers"):
        model.prefill(ids[:2], cache=cache, sequences=[1, 1])
    model.prefill(ids[:1], cache=cache, sequences=[1])
    with pytest.raises(ValueError, match="that is listed"):
        model.decode(ids[:, 0], cache, sequences=[1])
    with pytest.raises(ValueError, match="different numbers"):
        model.decode(ids[:1, 0], cache, sequences=[3])
    with pytest.raises(ValueError, match="empty cache"):
        model.prefill(ids, cache=cache)
    assert cache.lengths == [0, 5, 0]


@pytest.mark.gpu
def test_a_step_of_no_sequence_is_reported():
    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg = small()
    model = SharqDecoder(cfg, torch.device("cuda"), seed=3)
    ids = torch.randint(0, cfg.vocab, (2, 9), generator=torch.Generator().manual_seed(1)).cuda()
    cache = model.new_cache(2, 32, page_size=16)
    model.prefill(ids[:, :8], cache=cache)
    cache.reserve([1, 1])
    before = cache.k.view(torch.int16).clone()
    positions = torch.tensor([8, 8], dtype=torch.int32).cuda()
    logits = model.decode_step(ids[:, 8], cache, positions, positions + 1, weight_only=True, rows=torch.tensor([1, 2]).cuda())
    with pytest.raises(RuntimeError, match="paged cache"):
        ops.check_device_errors()
    assert bool(torch.isfinite(logits[0]).all()) and bool(logits[1].isnan().all())
    page = cache._held[1][0]  # only the other sequence's token went into the cache
    before[:, page, :, 8] = cache.k.view(torch.int16)[:, page, :, 8]
    assert torch.equal(cache.k.view(torch.int16), before)
