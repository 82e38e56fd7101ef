"""More operators of a serving step, as cases to be timed and compared.

Kinds of case (the `kind` of a case dict):

  prompt   attention of ragged prompts whose rows lie one behind the other, causal, with a sliding window and a few first tokens that stay
           visible (ops.prompt_attention); `before`: keys that every sequence already has ahead of its queries (a later piece of a prompt).
  token    attention of one new token per sequence over a paged cache, with a sliding window and first tokens that stay visible
           (ops.paged_attention with window and sinks).
  plan     pages and places for a step's tokens, handed out on the GPU from the sequences' lengths: ended sequences give their pages back, the
           others' new tokens get pages (ops.plan_paged_step).
  rules    penalties for repeated tokens, biases and grammar masks on logits (ops.adjust_logits).

window 0: none.  Head counts and vocabularies are those of the package's own configurations (32 / 8 heads of 128, 28 / 4 heads, one of eight
tensor-parallel ranks: 4 / 1; 128256, 152064 and 32000 tokens), or generic.
"""
import math

import torch

own = False

DEV = "cuda"
HEADS = ((32, 8), (28, 4), (4, 1), (8, 8), (16, 1))


def listed():
    return [
        # one short prompt: latency
        {"name": "prompt 1 x 200", "kind": "prompt", "seqs": 1, "rows": 200, "before": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 128, "sinks": 4},
        # ragged prompts of a batch under a narrow window
        {"name": "prompt 9 ragged", "kind": "prompt", "seqs": 9, "rows": 16001, "before": 0, "heads": 28, "kv_heads": 4, "dim": 128,
         "window": 1024, "sinks": 4},
        # a long document under a wide window
        {"name": "prompt 1 x 32768", "kind": "prompt", "seqs": 1, "rows": 32768, "before": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 4096, "sinks": 4},
        # a later piece of long prompts, all of whose keys stay visible, with heads of 64
        {"name": "prompt 2 pieces", "kind": "prompt", "seqs": 2, "rows": 4095, "before": 6000, "heads": 8, "kv_heads": 8, "dim": 64,
         "window": 0, "sinks": 0},
        # one user far into a conversation: latency
        {"name": "token 1 x 100000", "kind": "token", "seqs": 1, "shortest": 100000, "longest": 100000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "fp8": False, "window": 4096, "sinks": 4},
        # a decode batch of mixed lengths over a cache of 8-bit values, one of its rows empty
        {"name": "token 96 ragged e4m3", "kind": "token", "seqs": 96, "shortest": 0, "longest": 12000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "fp8": True, "window": 2048, "sinks": 16},
        # one of eight tensor-parallel ranks, pages of an odd size, first tokens that end inside a page
        {"name": "token 33 rank", "kind": "token", "seqs": 33, "shortest": 50, "longest": 9001, "heads": 4, "kv_heads": 1, "dim": 128,
         "page": 24, "fp8": False, "window": 1000, "sinks": 5},
        # a decode step of a small batch
        {"name": "plan 16 x 1", "kind": "plan", "seqs": 16, "longest": 1500, "prompts": 0, "ended": 0, "page": 16},
        # a step of a full server: most sequences go on by a token, some end, others begin with their prompts
        {"name": "plan 1000 mixed", "kind": "plan", "seqs": 1000, "longest": 3000, "prompts": 60, "ended": 60, "page": 64},
        # one user: latency
        {"name": "rules 1 x 128256", "kind": "rules", "rows": 1, "vocab": 128256, "history": 700, "bias": 0, "mask": False, "bf16": False},
        # a full decode batch with long histories, biases and grammar masks
        {"name": "rules 256 x 152064", "kind": "rules", "rows": 256, "vocab": 152064, "history": 6000, "bias": 40, "mask": True, "bf16": False},
        # logits of 16 bits, masks alone beside the penalties
        {"name": "rules 61 x 32000 bf16", "kind": "rules", "rows": 61, "vocab": 32000, "history": 2047, "bias": 0, "mask": True, "bf16": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("prompt", "token", "plan", "rules"))
    if kind == "plan":
        seqs = _log(rng, 1, 1000)
        ended = rng.choice((0, rng.randint(0, seqs // 4)))
        return {"kind": kind, "seqs": seqs, "longest": _log(rng, 1, 3000), "prompts": min(ended, rng.randint(0, 60)), "ended": ended,
                "page": rng.choice((8, 16, 24, 64, 128))}
    if kind == "rules":
        vocab = rng.choice((128256, 152064, 32000, _log(rng, 100, 152064)))
        return {"kind": kind, "rows": _log(rng, 1, 250), "vocab": vocab, "history": _log(rng, 1, 6000), "bias": rng.choice((0, _log(rng, 1, 80))),
                "mask": rng.random() < 0.5, "bf16": rng.random() < 0.3}
    heads, kv_heads = rng.choice(HEADS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice((64, 128, 128)),
            "window": rng.choice((0, _log(rng, 1, 4096), _log(rng, 64, 4096))), "sinks": rng.choice((0, 4, _log(rng, 1, 200)))}
    if kind == "prompt":
        seqs = _log(rng, 1, 24)
        rows = max(seqs, _log(rng, 1, 30000 if case["window"] else 8000))
        return {**case, "seqs": seqs, "rows": rows, "before": rng.choice((0, 0, _log(rng, 1, 4096)))}
    seqs = _log(rng, 1, 128)
    longest = _log(rng, 1, min(131072, (1 << 28) // (seqs * kv_heads * case["dim"])))
    return {**case, "seqs": seqs, "shortest": rng.randint(0, longest), "longest": longest, "page": rng.choice((8, 16, 24, 32, 64, 128)),
            "fp8": rng.random() < 0.4}


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, many small ones and few large ones."""
    return [hi if n == 1 else lo + int(round((hi - lo) * (i / (n - 1)) ** 2)) for i in range(n)]


def _prompt_rows(case):
    """Rows of every sequence of a `prompt` case: of unlike lengths that add up to its rows, one at least each."""
    n, total = case["seqs"], case["rows"]
    weights = [(i % 4 + 1) ** 2 for i in range(n)]
    rows = [1 + (total - n) * w // sum(weights) for w in weights]
    rows[-1] += total - sum(rows)
    return rows


def _visible(case, position):
    """How many keys a query at `position` sees."""
    window = case["window"] or position + 1
    near = min(window, position + 1)
    return near + min(case["sinks"], position + 1 - near)


def _scales(case, gen):
    if not case["fp8"]:
        return None
    return 0.02 + 0.02 * torch.rand(case["kv_heads"], generator=gen, device=DEV)


def _cache(pages, case, gen, scale):
    """A cache in use: keys or values N(0, 1) with some larger channels; scale: one per head for 8-bit values."""
    x = torch.randn((pages, case["kv_heads"], case["page"], case["dim"]), generator=gen, device=DEV, dtype=torch.bfloat16)
    x[..., ::29] *= 3
    if not case["fp8"]:
        return x
    return (x.float() / scale[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)


def _prepare_token(case, gen):
    """Lengths in random order, pages scattered over a cache with a few spare ones."""
    lengths = torch.tensor(_spread(case["seqs"], case["shortest"], case["longest"]), device=DEV, dtype=torch.int32)
    lengths = lengths[torch.randperm(case["seqs"], generator=gen, device=DEV)]
    counts = (lengths.long() + case["page"] - 1) // case["page"]
    pages, most = int(counts.sum()) + 3, max(1, int(counts.max()))
    at = torch.arange(most, device=DEV)
    table = torch.randperm(pages, generator=gen, device=DEV)[((counts.cumsum(0) - counts)[:, None] + at).clamp(max=pages - 1)]
    state = {"lengths": lengths, "table": torch.where(at < counts[:, None], table, 0).to(torch.int32).contiguous()}
    state["q"] = (1.5 * torch.randn(case["seqs"], case["heads"], case["dim"], generator=gen, device=DEV)).to(torch.bfloat16)
    for t in ("k", "v"):
        state[t + "_scale"] = _scales(case, gen)
        state[t + "_cache"] = _cache(pages, case, gen, state[t + "_scale"])
    return state


def _prepare_prompt(case, gen):
    """Queries and keys with some larger channels; values are the last columns of a merged activation, as the package's linears leave them."""
    rows = torch.tensor(_prompt_rows(case), device=DEV)
    keys = rows + case["before"]
    total, dim, kv_heads = int(keys.sum()), case["dim"], case["kv_heads"]
    q = torch.randn(case["rows"], case["heads"], dim, generator=gen, device=DEV, dtype=torch.bfloat16)
    k = torch.randn(total, kv_heads, dim, generator=gen, device=DEV, dtype=torch.bfloat16)
    q[..., ::29] *= 3
    k[..., ::31] *= 2
    merged = torch.randn(total, 2 * kv_heads * dim, generator=gen, device=DEV, dtype=torch.bfloat16)
    ends = [torch.cat((torch.zeros(1, device=DEV), n.cumsum(0))).to(torch.int32) for n in (rows, keys)]
    return {"q": q, "k": k, "v": merged[:, kv_heads * dim:].view(total, kv_heads, dim), "offsets": ends[0], "k_offsets": ends[1]}


def _prepare_plan(case, gen):
    """A server's sequences in mid-flight: lengths, page tables with room to grow, a stack of free pages, and what this step asks for."""
    seqs, page = case["seqs"], case["page"]
    lengths = torch.tensor(_spread(seqs, min(1, case["longest"]), case["longest"]), device=DEV)[torch.randperm(seqs, generator=gen, device=DEV)]
    held = (lengths + page - 1) // page
    most = 4 * (-(-case["longest"] // page) + 64)
    pages = seqs * most
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    at = torch.arange(most, device=DEV)
    table = torch.where(at < held[:, None], order[(held.cumsum(0) - held)[:, None] + at.clamp(max=most - 1)], 0).to(torch.int32)
    used = int(held.sum())
    stack = torch.cat((order[used:], order[:used]))  # what lies behind the free ones is stale
    counts = torch.ones(seqs, dtype=torch.int32, device=DEV)
    which = torch.randperm(seqs, generator=gen, device=DEV)[:case["ended"]]
    released = torch.zeros(seqs, dtype=torch.bool, device=DEV)
    released[which] = True
    counts[which] = 0
    counts[which[:case["prompts"]]] = torch.randint(1, case["longest"] + 1, (case["prompts"],), generator=gen, device=DEV, dtype=torch.int32)
    return {"lengths": lengths.to(torch.int32), "table": table.contiguous(), "stack": stack, "free": torch.tensor([pages - used], dtype=torch.int32, device=DEV),
            "counts": counts, "released": released, "rows": seqs + case["prompts"] * case["longest"]}


def _prepare_rules(case, gen):
    """Logits N(0, 3); histories of which half is the prompt, common tokens far more often than rare ones; masks that leave a few tokens in a
    hundred, or most of them."""
    rows, vocab, width = case["rows"], case["vocab"], case["history"]
    logits = 3 * torch.randn(rows, vocab, generator=gen, device=DEV)
    tokens = (torch.exp(torch.rand(rows, width, generator=gen, device=DEV) * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1)
    lengths = torch.tensor(_spread(rows, width // 3, width), device=DEV, dtype=torch.int32)
    state = {"logits": logits.to(torch.bfloat16) if case["bf16"] else logits, "tokens": tokens.to(torch.int32), "lengths": lengths,
             "prompt_lengths": lengths // 2, "bias": None, "mask": None}
    state["repetition"] = 1 + 0.5 * torch.rand(rows, generator=gen, device=DEV)
    state["presence"] = torch.rand(rows, generator=gen, device=DEV)
    state["frequency"] = 0.3 * torch.rand(rows, generator=gen, device=DEV)
    if case["bias"]:
        offsets = torch.arange(rows + 1, device=DEV, dtype=torch.int32) * case["bias"]
        ids = torch.randint(0, vocab, (rows * case["bias"],), generator=gen, device=DEV, dtype=torch.int32)
        state["bias"] = (offsets, ids, 4 * torch.randn(rows * case["bias"], generator=gen, device=DEV))
    if case["mask"]:
        keep = torch.where(torch.arange(rows, device=DEV) % 3 == 0, 0.97, 0.02)
        words = -(-vocab // 32)
        bits = torch.rand(rows, words, 32, generator=gen, device=DEV) < keep[:, None, None]
        bits[:, 0, 0] = True
        state["mask"] = (bits.long() << torch.arange(32, device=DEV)).sum(-1).to(torch.int32)
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    make = {"prompt": _prepare_prompt, "token": _prepare_token, "plan": _prepare_plan, "rules": _prepare_rules}[case["kind"]]
    return {"case": case, **make(case, gen)}


# --------------------------------------------------------------------------- plain forms

def _softmax_product(scores, seen, v):
    """Softmax of the scores where `seen`, times v; zeros for a row that sees nothing."""
    scores = torch.where(seen, scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - torch.where(top == -torch.inf, 0, top)), 0)
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, (p @ v) / total, 0)


def _prompt(s):
    """Query rows of a sequence in pieces, so that the scores fit the memory, each with the keys that some row of it may see."""
    case = s["case"]
    heads, kv_heads, dim, piece = case["heads"], case["kv_heads"], case["dim"], 1024
    out = torch.empty_like(s["q"])
    q0 = k0 = 0
    for rows in _prompt_rows(case):
        keys = rows + case["before"]
        k, v = (s[t][k0:k0 + keys].float().transpose(0, 1) for t in ("k", "v"))
        for a in range(0, rows, piece):
            b = min(rows, a + piece)
            at = torch.arange(case["before"] + a, case["before"] + b, device=DEV)[:, None]
            first = max(0, case["before"] + a + 1 - case["window"]) if case["window"] else 0
            skip = min(case["sinks"], first)
            j = torch.cat((torch.arange(skip, device=DEV), torch.arange(first, case["before"] + b, device=DEV)))
            kj, vj = (torch.cat((x[:, :skip], x[:, first:case["before"] + b]), 1) for x in (k, v))
            seen = j <= at
            if case["window"]:
                seen = seen & ((at - j < case["window"]) | (j < case["sinks"]))
            q = s["q"][q0 + a:q0 + b].float().view(b - a, kv_heads, heads // kv_heads, dim).permute(1, 2, 0, 3)
            got = _softmax_product(q @ kj[:, None].transpose(2, 3) * dim ** -0.5, seen, vj[:, None])
            out[q0 + a:q0 + b] = got.permute(2, 0, 1, 3).reshape(b - a, heads, dim).to(torch.bfloat16)
        q0, k0 = q0 + rows, k0 + keys
    return out


def _token(s):
    """The visible tokens of every sequence gathered from its pages: the first ones, then the window's."""
    case = s["case"]
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    near = min(case["window"] or case["longest"], case["longest"])
    first = min(case["sinks"] if case["window"] else 0, case["longest"])
    n = s["lengths"].long()[:, None]
    begin = (n - near).clamp(min=0)
    j = torch.cat((torch.arange(first, device=DEV).expand(case["seqs"], first), begin + torch.arange(near, device=DEV)), 1)
    seen = (j < n) & ((torch.arange(first + near, device=DEV) >= first) | (j < begin))
    j = j.clamp(max=max(0, case["longest"] - 1))
    pages, slots = s["table"].long().gather(1, j // page), j % page

    def gathered(cache, scale):
        held = (cache if scale is None else cache.view(torch.uint8))[pages, :, slots]
        x = (held if scale is None else held.view(cache.dtype)).float().transpose(1, 2)
        return x if scale is None else x * scale[:, None, None]

    q = s["q"].float().view(case["seqs"], kv_heads, case["heads"] // kv_heads, dim)
    scores = q @ gathered(s["k_cache"], s["k_scale"]).transpose(2, 3) * dim ** -0.5
    v = torch.where(seen[:, None, :, None], gathered(s["v_cache"], s["v_scale"]), 0)
    return _softmax_product(scores, seen[:, None, None], v).view(case["seqs"], case["heads"], dim).to(torch.bfloat16)


def _plan(s):
    """Everything from prefix sums over the sequences; the state's table, lengths and stack are the step's results too."""
    page, most, rows = s["case"]["page"], s["table"].shape[1], s["rows"]
    at = torch.arange(most, device=DEV)
    # ended sequences put their pages back, the last page first
    length = s["lengths"].long()
    back = torch.where(s["released"], (length + page - 1) // page, 0)
    to = s["free"].long() + (back.cumsum(0) - back)[:, None] + back[:, None] - 1 - at
    to = torch.where(at < back[:, None], to, s["stack"].numel())
    stack = torch.cat((s["stack"], s["stack"][:1])).scatter(0, to.view(-1), s["table"].view(-1))[:-1]
    free = s["free"].long() + back.sum()
    length = torch.where(s["released"], 0, length)
    # new tokens, and the pages they need beyond those held
    counts = s["counts"].long()
    held = (length + page - 1) // page
    need = (length + counts + page - 1) // page - held
    taken = need.cumsum(0)
    ends = counts.cumsum(0)
    given = ((need == 0) | (taken <= free)) & (ends <= rows)
    new = given[:, None] & (at >= held[:, None]) & (at < (held + need)[:, None])
    place = free - 1 - ((taken - need)[:, None] + at - held[:, None])
    table = torch.where(new, stack[place.clamp(0, stack.numel() - 1)], s["table"])
    # every row's sequence and position
    r = torch.arange(rows, device=DEV)
    i = torch.searchsorted(ends, r, right=True)
    there = i < ends.numel()
    i = i.clamp(max=ends.numel() - 1)
    positions = torch.where(there & given[i], length[i] + r - (ends - counts)[i], -1)
    s["table"].copy_(table)
    s["stack"].copy_(stack)
    s["lengths"].copy_(length + torch.where(given, counts, 0))
    s["free"].copy_(free - torch.where(given, need, 0).sum())
    offsets = torch.cat((torch.zeros_like(ends[:1]), ends)).to(torch.int32)
    return offsets, positions.to(torch.int32), torch.where(there, i, 0).to(torch.int32)


def _rules(s):
    """Arithmetic in 64 bits: a penalty or a bias may leave little of a logit."""
    rows, vocab = s["logits"].shape
    x = s["logits"].double()
    at = torch.arange(s["tokens"].shape[1], device=DEV)
    live, fresh = at < s["lengths"][:, None], at >= s["prompt_lengths"][:, None]
    ids = s["tokens"].long()
    seen = torch.zeros(rows, vocab, dtype=torch.int32, device=DEV).scatter_add_(1, ids, live.int()) > 0
    count = torch.zeros(rows, vocab, dtype=torch.int32, device=DEV).scatter_add_(1, ids, (live & fresh).int())
    r, p, f = (s[t].double()[:, None] for t in ("repetition", "presence", "frequency"))
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - f * count - torch.where(count > 0, p, 0)
    if s["bias"] is not None:
        offsets, bias_ids, values = s["bias"]
        row = torch.searchsorted(offsets, torch.arange(bias_ids.numel(), device=DEV, dtype=torch.int32), right=True) - 1
        x = x.index_put((row, bias_ids.long()), values.double(), accumulate=True)
    if s["mask"] is not None:
        keep = (s["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        x = torch.where(keep.flatten(1)[:, :vocab] != 0, x, -torch.inf)
    return x.to(s["logits"].dtype)


def run(state):
    case = state["case"]
    window = case.get("window") or None
    if own:
        from sharq_b200 import ops

        if case["kind"] == "prompt":
            return ops.prompt_attention(state["q"], state["k"], state["v"], state["offsets"], window=window, sinks=case["sinks"],
                                        k_offsets=state["k_offsets"] if case["before"] else None)
        if case["kind"] == "token":
            return ops.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["table"], state["lengths"],
                                       k_scale=state["k_scale"], v_scale=state["v_scale"], window=window, sinks=case["sinks"])
        if case["kind"] == "plan":
            got = ops.plan_paged_step(state["table"], state["lengths"], state["counts"], state["stack"], state["free"], case["page"],
                                      state["rows"], released=state["released"])
        else:
            return ops.adjust_logits(state["logits"], state["tokens"], state["lengths"], prompt_lengths=state["prompt_lengths"],
                                     repetition=state["repetition"], presence=state["presence"], frequency=state["frequency"],
                                     bias=state["bias"], mask=state["mask"])
    else:
        got = {"prompt": _prompt, "token": _token, "plan": _plan, "rules": _rules}[case["kind"]](state)
    if case["kind"] != "plan":
        return got
    return {"offsets": got[0], "positions": got[1], "sequences": got[2], "table": state["table"], "lengths": state["lengths"],
            "stack": state["stack"], "free": state["free"]}


def work(case):
    if case["kind"] == "plan":
        # the sequences' numbers, and the rows' places; of the pages as many as change hands, about
        rows = case["seqs"] + case["prompts"] * case["longest"]
        moved = (case["ended"] + case["prompts"]) * (case["longest"] // 2) // case["page"]
        return {"bytes": case["seqs"] * (4 + 4 + 1 + 4 + 4) + 8 * rows + 8 * moved, "flops": 8 * case["seqs"]}
    if case["kind"] == "rules":
        size, cells = 2 if case["bf16"] else 4, case["rows"] * case["vocab"]
        history = sum(_spread(case["rows"], case["history"] // 3, case["history"]))
        return {"bytes": 2 * size * cells + 4 * history + 8 * case["rows"] * case["bias"] + (cells // 8 if case["mask"] else 0),
                "flops": 4 * history + cells}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "prompt":
        counts, before = _prompt_rows(case), case["before"]
        pairs = sum(_visible(case, before + i) for n in counts for i in range(n))
        keys = sum(counts) + before * len(counts)
        return {"bytes": 2 * dim * (2 * case["rows"] * heads + 2 * keys * kv_heads), "flops": 4 * pairs * heads * dim}
    tokens = sum(_visible(case, n - 1) for n in _spread(case["seqs"], case["shortest"], case["longest"]) if n > 0)
    return {"bytes": tokens * kv_heads * dim * 2 * (1 if case["fp8"] else 2) + 2 * case["seqs"] * heads * dim * 2, "flops": 4 * tokens * heads * dim}


# --------------------------------------------------------------------------- from the definitions, in 64 bits

def _seen64(case, p, j):
    """Whether the query at p sees the key at j."""
    near = (p - j < case["window"]) if case["window"] else torch.ones_like(p - j, dtype=torch.bool)
    return (j <= p) & (near | (j < case["sinks"]))


def _weighted64(q, k, v, seen):
    """Rows of q [n, dim] over the keys that they see, in 64 bits."""
    a = (q @ k.T / math.sqrt(q.shape[1])).masked_fill(~seen, -math.inf)
    return torch.softmax(a, -1).nan_to_num(0.0) @ v


def _prompt64(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    group = case["heads"] // case["kv_heads"]
    starts, key_starts = s["offsets"].tolist(), s["k_offsets"].tolist()
    for i in range(case["seqs"]):
        rows, keys = slice(starts[i], starts[i + 1]), slice(key_starts[i], key_starts[i + 1])
        for h in range(case["kv_heads"]):
            k, v = s["k"][keys, h].double(), s["v"][keys, h].double()
            for r in range(rows.start, rows.stop, 2048):
                end = min(rows.stop, r + 2048)
                p = case["before"] + torch.arange(r - rows.start, end - rows.start, device=DEV)
                # the keys ahead of the piece's window are seen by none of its rows, but for the first ones
                cut = max(case["sinks"], int(p[0]) + 1 - case["window"]) if case["window"] else 0
                j = torch.arange(k.shape[0], device=DEV)
                j = j[(j < case["sinks"]) | (j >= cut)] if case["window"] else j
                j = j[j <= p[-1]]
                seen = _seen64(case, p[:, None], j)
                for g in range(h * group, h * group + group):
                    out[r:end, g] = _weighted64(s["q"][r:end, g].double(), k[j], v[j], seen)
    return out


def _token64(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    group = case["heads"] // case["kv_heads"]
    for i, n in enumerate(s["lengths"].tolist()):
        j = torch.arange(n, device=DEV)
        j = j[_seen64(case, torch.tensor(n - 1, device=DEV), j)]
        pages, slots = s["table"][i].long()[j // case["page"]], j % case["page"]
        for h in range(case["kv_heads"] if n else 0):
            k, v = ((s[c].view(torch.uint8) if case["fp8"] else s[c])[pages, h, slots] for c in ("k_cache", "v_cache"))
            if case["fp8"]:
                k, v = (x.view(torch.float8_e4m3fn).double() * s[c][h].double() for x, c in ((k, "k_scale"), (v, "v_scale")))
            heads = slice(h * group, h * group + group)
            out[i, heads] = _weighted64(s["q"][i, heads].double(), k.double(), v.double(), torch.ones(1, len(j), dtype=torch.bool, device=DEV))
    return out


def _rules64(case, s):
    out = s["logits"].double()
    for i in range(case["rows"]):
        history = s["tokens"][i, :int(s["lengths"][i])].long()
        seen, counts = history.unique(), torch.bincount(history[int(s["prompt_lengths"][i]):], minlength=case["vocab"])
        x = out[i, seen]
        r = s["repetition"][i].double()
        out[i, seen] = torch.where(x > 0, x / r, x * r)
        made = counts.nonzero()[:, 0]
        out[i, made] -= s["frequency"][i].double() * counts[made] + s["presence"][i].double()
        if s["bias"] is not None:
            offsets, ids, values = s["bias"]
            part = slice(int(offsets[i]), int(offsets[i + 1]))
            out[i].index_add_(0, ids[part].long(), values[part].double())
        if s["mask"] is not None:
            token = torch.arange(case["vocab"], device=DEV)
            out[i, (s["mask"][i].long()[token // 32] >> (token % 32)) & 1 == 0] = -math.inf
    return out


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s = prepare(case, seed)
    return {"prompt": _prompt64, "token": _token64, "rules": _rules64}[case["kind"]](case, s)
