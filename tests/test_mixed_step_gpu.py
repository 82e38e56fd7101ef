"""A server's step with prompts and single tokens in it: the operators in the order in which a server calls them, each against its definition."""
import pytest
import torch

from sharq_b200 import ops
from tests import paged_util as P
from tests.test_logit_rules_gpu import check as check_logits, rules64
from tests.test_prompt_attention_gpu import bound as prompt_bound, definition64 as prompt64
from tests.test_windowed_attention_gpu import definition64 as token64

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page,window,sinks", [(16, 30, 4), (24, None, 0), (64, 1000, 3)])
def test_prompts_beside_single_tokens(page, window, sinks):
    """What is left of a sequence from step to step is its pages: of every row the result is that of its whole sequence."""
    seqs, heads, kv, dim, most, vocab = 6, 8, 2, 128, 10, 1000
    g = torch.Generator(device="cuda").manual_seed(page)
    pages = seqs * most
    table, lengths, stack, free = i32([[-1] * most] * seqs), i32([0] * seqs), torch.arange(pages, device="cuda", dtype=torch.int32), i32([pages])
    k_cache, v_cache, *_ = P.make_cache(pages, kv, page, dim, False, 2)
    cos, sin = P.rope_tables(most * page, dim)
    history, held = torch.full((seqs, 64), -1, dtype=torch.int32, device="cuda"), i32([0] * seqs)
    head = torch.randn(heads * dim, vocab, generator=g, device="cuda") / 32
    seen = dict(window=window, sinks=sinks) if window else {}

    # tokens of every sequence, and those that end first
    for counts, released in (([7, 0, 90, 33, 1, 0], []), ([1, 41, 1, 1, 0, 16], []), ([1, 1, 60, 0, 1, 1], [2]), ([1, 1, 1, 1, 1, 1], []), ([0, 130, 1, 1, 5, 1], [1, 4]),
                             ([1, 1, 1, 1, 1, 1], [])):
        before = [0 if i in released else n for i, n in enumerate(lengths.tolist())]
        going = torch.tensor([i for i in range(seqs) if before[i] > 0 and counts[i] == 1], dtype=torch.long, device="cuda")
        rows = sum(counts) + 3
        qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g, device="cuda").to(torch.bfloat16)
        v = qkv[:, (heads + kv) * dim:].view(rows, kv, dim)

        ended = torch.zeros(seqs, dtype=torch.bool, device="cuda")
        ended[released] = True
        offsets, positions, which = ops.plan_paged_step(table, lengths, i32(counts), stack, free, page, rows, released=ended, strict=True)
        q, k = ops.rope_append_paged(qkv, heads, kv, dim, cos, sin, positions, table, k_cache, v_cache, sequences=which, return_k=True)
        out = ops.prompt_attention(q, k, v, offsets, **seen)
        if going.numel() > 0:
            at = offsets[going].long()
            out[at] = ops.paged_attention(q[at], k_cache, v_cache, table[going], lengths[going], **seen)
        last = (offsets[1:] - 1).clamp(min=0).long()
        logits = out[last].flatten(1).float() @ head
        rules = dict(tokens=history, lengths=held, presence=torch.full((seqs,), 0.5, device="cuda"), repetition=torch.full((seqs,), 1.2, device="cuda"))
        chosen = ops.adjust_logits(logits, **rules)

        ops.check_device_errors()
        assert lengths.tolist() == [n + c for n, c in zip(before, counts)]
        assert (out[sum(counts):] == 0).all()
        start = offsets.tolist()
        for i, n in enumerate(counts):
            part = slice(start[i], start[i] + n)
            assert positions[part].tolist() == list(range(before[i], before[i] + n)) and (which[part] == i).all()
            if before[i] > 0 and n == 1:
                want, size, reach = token64(q[part], k_cache.double(), v_cache.double(), table[i:i + 1], [before[i] + 1], window or 10 ** 6, sinks, dim ** -0.5)
                limit = P.attention_bound(want, size, reach, dim, before[i] + 1, False)
            elif n > 0:
                want, size, reach = prompt64(q[part], k[part], v[part], [n], [n], window or 0, sinks, dim ** -0.5)
                limit = prompt_bound(want, size, reach, dim, n)
                where = torch.arange(n, device="cuda")
                kept = table[i].long()[where // page], slice(None), where % page
                assert torch.equal(k_cache[kept], k[part]) and torch.equal(v_cache[kept], v[part])
            else:
                continue
            assert ((out[part].double() - want).abs() <= limit).all()
        check_logits(logits, chosen, rules64(logits, **rules))
        token = chosen.argmax(-1).int()
        for i, n in enumerate(counts):
            if n > 0:
                history[i, held[i]] = token[i]
                held[i] += 1
    assert len(set(table[s, j].item() for s in range(seqs) for j in range(-(-int(lengths[s]) // page)))) == pages - int(free)
