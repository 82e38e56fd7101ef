"""The operators of a decode step, as cases to be timed and compared.

Kinds of case (the `kind` of a case dict):

  append   rotary embedding of the query and key heads of a merged qkv activation, with keys and values
           appended to a paged cache (ops.rope_append_paged).  seqs == rows: one token of every sequence; fewer seqs:
           the rows of ragged prompts, sequence after sequence, from position `start` on.
  attend   attention of one new token per sequence over its part of a paged cache (ops.paged_attention), lengths
           from `shortest` to `longest`, most of them short.
  matvec   product of a few unquantised activation rows with a 4-bit weight with one scale per 16 elements of K
           (ops.weight_only_linear), in the buffers of a quantised linear.

Head counts and projections are those of the package's own configurations (32 / 8 heads of 128, 28 / 4 heads, one of eight
tensor-parallel ranks: 4 / 1), or generic.
"""
import math

import torch

own = False

DEV = "cuda"
THETA = 5e5
HEADS = ((32, 8), (28, 4), (4, 1), (8, 8), (16, 1))
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # the first token after a short prompt, a single user: latency
        {"name": "append 1", "kind": "append", "rows": 1, "seqs": 1, "start": 517, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "fp8": False, "return_k": False},
        # a full decode batch into a cache of 8-bit values
        {"name": "append 256 e4m3", "kind": "append", "rows": 256, "seqs": 256, "start": 900, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "fp8": True, "return_k": False},
        # ragged prompts, whose attention also reads the rotated keys
        {"name": "append prompts 16384", "kind": "append", "rows": 16384, "seqs": 7, "start": 0, "heads": 28, "kv_heads": 4,
         "dim": 128, "page": 64, "fp8": False, "return_k": True},
        # one user, a short conversation: latency
        {"name": "attend 1 x 97", "kind": "attend", "seqs": 1, "shortest": 97, "longest": 97, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "fp8": False},
        # one user, a long document
        {"name": "attend 1 x 131072", "kind": "attend", "seqs": 1, "shortest": 131072, "longest": 131072, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "fp8": False},
        # a decode batch of mixed lengths, one of its rows empty
        {"name": "attend 64 ragged", "kind": "attend", "seqs": 64, "shortest": 0, "longest": 8191, "heads": 28, "kv_heads": 4,
         "dim": 128, "page": 32, "fp8": False},
        # a large batch over a cache of 8-bit values
        {"name": "attend 128 ragged e4m3", "kind": "attend", "seqs": 128, "shortest": 33, "longest": 8192, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "fp8": True},
        # one of eight tensor-parallel ranks: a single key/value head
        {"name": "attend 5 rank", "kind": "attend", "seqs": 5, "shortest": 1000, "longest": 20011, "heads": 4, "kv_heads": 1,
         "dim": 128, "page": 128, "fp8": False},
        # the projections of one token, and of small decode batches
        {"name": "matvec 1 o_proj", "kind": "matvec", "rows": 1, "n": 4096, "k": 4096, "bias": False},
        {"name": "matvec 1 gate_up", "kind": "matvec", "rows": 1, "n": 28672, "k": 4096, "bias": False},
        {"name": "matvec 8 down", "kind": "matvec", "rows": 8, "n": 4096, "k": 14336, "bias": False},
        {"name": "matvec 13 qkv bias", "kind": "matvec", "rows": 13, "n": 4608, "k": 3584, "bias": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "matvec"))
    if kind == "matvec":
        return {"kind": kind, "rows": rng.randint(1, 16), "n": _log(rng, 64, 28672), "k": 64 * _log(rng, 2, 224),
                "bias": rng.random() < 0.5}
    heads, kv_heads = rng.choice(HEADS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice((64, 128, 128)),
            "page": rng.choice((8, 16, 24, 32, 64, 128)), "fp8": rng.random() < 0.4}
    if kind == "append":
        seqs = _log(rng, 1, 256)
        rows = seqs if rng.random() < 0.5 else max(seqs, _log(rng, 1, 16384))
        return {**case, "rows": rows, "seqs": seqs, "start": rng.choice((0, _log(rng, 1, 1500))), "return_k": rng.random() < 0.5}
    seqs = _log(rng, 1, 192)
    longest = _log(rng, 1, min(131072, (1 << 29) // (seqs * kv_heads * case["dim"])))
    return {**case, "seqs": seqs, "shortest": rng.randint(0, longest), "longest": longest}


def _lengths(case):
    """Lengths of the sequences of an `attend` case, shortest first: many short ones and few long ones."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    return [hi if n == 1 else lo + int(round((hi - lo) * (i / (n - 1)) ** 2)) for i in range(n)]


def _prompt_rows(case):
    """Rows of every sequence of an `append` case."""
    return [case["rows"] // case["seqs"] + (i < case["rows"] % case["seqs"]) for i in range(case["seqs"])]


def _page_table(lengths, page, gen):
    """Every sequence's pages, scattered over a cache with a few spare ones: (table [seqs, most], pages of the cache)."""
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    most = max(1, max(counts))
    firsts = torch.tensor([sum(counts[:i]) for i in range(len(counts))], device=DEV)
    held = torch.tensor(counts, device=DEV)
    at = torch.arange(most, device=DEV)
    table = order[(firsts[:, None] + at).clamp(max=pages - 1)]
    return torch.where(at < held[:, None], table, torch.zeros_like(table)).contiguous(), pages


def _cache(pages, case, gen, scale):
    """A cache in use: keys or values N(0, 1) with some larger channels; scale: one per head for 8-bit values."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.bfloat16)
    x[..., ::29] *= 3
    if not case["fp8"]:
        return x
    return (x.float() / scale[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)


def _scales(case, gen):
    if not case["fp8"]:
        return None
    return 0.02 + 0.02 * torch.rand(case["kv_heads"], generator=gen, device=DEV)


def _weight(n, k, gen):
    """A weight N(0, 0.02) as the package's linears hold it: e2m1 codes two to a byte, element 2i in the low half; per 16
    elements of a row a UE4M3 scale, in tiles of 128 rows x 4 scales (row r % 32 apart by 16 bytes, r / 32 % 4 by 4); a scale of the tensor."""
    w = 0.02 * torch.randn(n, k, generator=gen, device=DEV)
    scale = (w.abs().max() / (448.0 * 6.0)).clamp(min=1e-9)
    groups = (w / scale).view(n, k // 16, 16)
    sf = (groups.abs().amax(-1) / 6.0).clamp(2.0 ** -9, 448.0).to(torch.float8_e4m3fn)
    groups = groups / sf.float()[..., None]
    steps = torch.tensor([(a + b) / 2 for a, b in zip(E2M1, E2M1[1:])], device=DEV)
    codes = torch.bucketize(groups.abs(), steps).to(torch.uint8) + 8 * (groups < 0).to(torch.uint8)
    codes = codes.view(n, k // 2, 2)
    q = codes[..., 0] + 16 * codes[..., 1]
    rows = (n // 128 + 1) * 128
    padded = torch.zeros(rows, k // 16, dtype=torch.uint8, device=DEV)
    padded[:n] = sf.view(torch.uint8)
    tiles = padded.view(rows // 128, 4, 32, k // 64, 4).permute(0, 3, 2, 1, 4)
    return q.contiguous(), tiles.contiguous().view(-1), scale.float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "matvec":
        q, sf, scale = _weight(case["n"], case["k"], gen)
        x = torch.randn(case["rows"], case["k"], generator=gen, device=DEV)
        x[:, ::97] *= 20  # outlier channels
        bias = (0.02 * torch.randn(case["n"], generator=gen, device=DEV)).to(torch.bfloat16) if case["bias"] else None
        return {"case": case, "x": x.to(torch.bfloat16), "q": q, "sf": sf, "scale": scale, "bias": bias,
                "lut": torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)}
    state = {"case": case, "k_scale": _scales(case, gen), "v_scale": _scales(case, gen)}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        counts = _prompt_rows(case)
        reach = [case["start"] + n for n in counts]
        rows = torch.tensor(counts, device=DEV)
        state["qkv"] = torch.randn(case["rows"], (heads + 2 * kv_heads) * dim, generator=gen, device=DEV, dtype=torch.bfloat16)
        state["sequences"] = torch.repeat_interleave(torch.arange(case["seqs"], device=DEV), rows).to(torch.int32)
        first = torch.repeat_interleave(rows.cumsum(0) - rows, rows)
        state["positions"] = (case["start"] + torch.arange(case["rows"], device=DEV) - first).to(torch.int32)
        angles = torch.outer(torch.arange(max(reach), device=DEV, dtype=torch.float64),
                             THETA ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim))
        angles = torch.cat((angles, angles), -1)
        state["cos"], state["sin"] = angles.cos().to(torch.bfloat16), angles.sin().to(torch.bfloat16)
    else:
        reach = _lengths(case)
        lengths = torch.tensor(reach, device=DEV, dtype=torch.int32)[torch.randperm(case["seqs"], generator=gen, device=DEV)]
        reach = lengths.tolist()
        state["lengths"] = lengths
        state["q"] = (1.5 * torch.randn(case["seqs"], heads, dim, generator=gen, device=DEV)).to(torch.bfloat16)
    state["table"], pages = _page_table(reach, case["page"], gen)
    state["k_cache"], state["v_cache"] = _cache(pages, case, gen, state["k_scale"]), _cache(pages, case, gen, state["v_scale"])
    return state


# --------------------------------------------------------------------------- plain forms

def _store(cache, pages, slots, x, scale):
    """x [rows, kv_heads, dim] into its places in a cache."""
    if scale is None:
        cache[pages, :, slots] = x.to(cache.dtype)
    else:
        cache.view(torch.uint8)[pages, :, slots] = (x / scale[:, None]).clamp(-448, 448).to(cache.dtype).view(torch.uint8)


def _append(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    rows, page = case["rows"], case["page"]
    position = s["positions"].long()
    x = s["qkv"].float().view(rows, heads + 2 * kv_heads, dim)
    cos, sin = s["cos"].float()[position][:, None], s["sin"].float()[position][:, None]
    qk, v = x[:, :heads + kv_heads], x[:, heads + kv_heads:]
    turned = torch.cat((-qk[..., dim // 2:], qk[..., :dim // 2]), -1)
    qk = qk * cos + turned * sin
    pages, slots = s["table"][s["sequences"].long(), position // page].long(), position % page
    _store(s["k_cache"], pages, slots, qk[:, heads:], s["k_scale"])
    _store(s["v_cache"], pages, slots, v, s["v_scale"])
    q = qk[:, :heads].to(torch.bfloat16)
    out = {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return {**out, "k": qk[:, heads:].to(torch.bfloat16)} if case["return_k"] else out


def _gathered(cache, table, scale):
    """A cache's pages in the order of their sequences, as float [seqs, kv_heads, tokens, dim]."""
    held = (cache if scale is None else cache.view(torch.uint8))[table.long()]
    x = (held if scale is None else held.view(cache.dtype)).float().transpose(1, 2).flatten(2, 3)
    return x if scale is None else x * scale[:, None, None]


def _attend(s):
    case = s["case"]
    kv_heads, dim = case["kv_heads"], case["dim"]
    k = _gathered(s["k_cache"], s["table"], s["k_scale"])
    tokens = k.shape[2]
    live = (torch.arange(tokens, device=DEV) < s["lengths"][:, None])[:, None, None]
    q = s["q"].float().view(case["seqs"], kv_heads, case["heads"] // kv_heads, dim)
    scores = torch.where(live, (q @ k.transpose(2, 3)) * dim ** -0.5, -torch.inf)
    del k
    top = scores.amax(-1, keepdim=True)
    p = torch.where(live, torch.exp(scores - top), 0)
    total = p.sum(-1, keepdim=True)
    v = torch.where(live.transpose(2, 3), _gathered(s["v_cache"], s["table"], s["v_scale"]), 0)
    out = torch.where(total > 0, (p @ v) / total, 0)
    return out.view(case["seqs"], case["heads"], dim).to(torch.bfloat16)


def _unpacked(s):
    """The 4-bit weight as float [n, k], without the scale of the tensor."""
    n, k = s["case"]["n"], s["case"]["k"]
    codes = torch.stack((s["q"] & 15, s["q"] >> 4), -1).view(n, k)
    rows = (n // 128 + 1) * 128
    sf = s["sf"].view(rows // 128, k // 64, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rows, k // 16)[:n]
    return (s["lut"][codes.int()].view(n, k // 16, 16) * sf.contiguous().view(torch.float8_e4m3fn).float()[..., None]).view(n, k)


def _matvec(s):
    y = (s["x"].float() @ _unpacked(s).T) * s["scale"]
    return (y if s["bias"] is None else y + s["bias"].float()).to(torch.bfloat16)


def run(state):
    case = state["case"]
    if own:
        from sharq_b200 import ops

        if case["kind"] == "append":
            got = ops.rope_append_paged(
                state["qkv"], case["heads"], case["kv_heads"], case["dim"], state["cos"], state["sin"], state["positions"],
                state["table"], state["k_cache"], state["v_cache"],
                sequences=None if case["rows"] == case["seqs"] else state["sequences"], k_scale=state["k_scale"],
                v_scale=state["v_scale"], return_k=case["return_k"])
            q, k = got if case["return_k"] else (got, None)
            out = {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
            return {**out, "k": k} if case["return_k"] else out
        if case["kind"] == "attend":
            return ops.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["table"], state["lengths"],
                                       k_scale=state["k_scale"], v_scale=state["v_scale"])
        return ops.weight_only_linear(state["x"], state["q"], state["sf"], state["scale"], bias=state["bias"])
    return {"append": _append, "attend": _attend, "matvec": _matvec}[case["kind"]](state)


def work(case):
    if case["kind"] == "matvec":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * k // 2 + n * k // 16 + 2 * m * (n + k) + 2 * n * case["bias"], "flops": 2 * m * n * k}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    size = 1 if case["fp8"] else 2
    if case["kind"] == "append":
        rows = case["rows"]
        read = rows * (heads + 2 * kv_heads) * dim * 2 + 2 * 2 * dim * max(_prompt_rows(case))
        return {"bytes": read + rows * dim * (2 * heads + 2 * kv_heads * size + 2 * kv_heads * case["return_k"]),
                "flops": 3 * rows * (heads + kv_heads) * dim}
    tokens = sum(_lengths(case))
    return {"bytes": tokens * kv_heads * dim * 2 * size + 2 * case["seqs"] * heads * dim * 2, "flops": 4 * tokens * heads * dim}


# --------------------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "matvec":
        n, k = case["n"], case["k"]
        value = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=DEV)
        row, group = torch.arange(n, device=DEV)[:, None], torch.arange(k // 16, device=DEV)[None]
        at = (row // 128) * (k // 64) * 512 + (group // 4) * 512 + (row % 32) * 16 + (row // 32 % 4) * 4 + group % 4
        sf = s["sf"].view(torch.float8_e4m3fn).double()[at]
        y = torch.zeros(case["rows"], n, dtype=torch.float64, device=DEV)
        x = s["x"].double().view(case["rows"], k // 16, 16)
        for i in range(16):  # element i of every group
            byte = s["q"].view(n, k // 16, 8)[..., i // 2]
            y += x[..., i] @ (value[(byte >> 4 if i % 2 else byte & 15).long()] * sf).T
        y = y * s["scale"].double()
        return y if s["bias"] is None else y + s["bias"].double()
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    table = s["table"].tolist()
    if case["kind"] == "append":
        x = s["qkv"].double().view(case["rows"], -1, 2, dim // 2)
        at = s["positions"].long()
        cos, sin = (s[t].double()[at].view(case["rows"], 1, 2, dim // 2) for t in ("cos", "sin"))
        a, b = x[:, :, 0], x[:, :, 1]
        turned = torch.stack((a * cos[:, :, 0] - b * sin[:, :, 0], b * cos[:, :, 1] + a * sin[:, :, 1]), 2).flatten(2)
        k, v = turned[:, heads:heads + kv_heads], x[:, heads + kv_heads:].flatten(2)
        caches = {}
        for name, new, scale in (("k_cache", k, s["k_scale"]), ("v_cache", v, s["v_scale"])):
            held = s[name].double()
            new = new if scale is None else new / scale.double()[:, None]
            new = new if scale is None else new.clamp(-448, 448)
            first = 0
            for i, n in enumerate(_prompt_rows(case)):
                spot = torch.arange(case["start"], case["start"] + n, device=DEV)
                held[s["table"][i].long()[spot // page], :, spot % page] = new[first:first + n]
                first += n
            caches[name] = held
        out = {"q": turned[:, :heads], **caches}
        return {**out, "k": k} if case["return_k"] else out
    out = torch.zeros(case["seqs"], heads, dim, dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        pages = torch.tensor(table[i][:-(-n // page)], device=DEV)
        k, v = ((s[c].view(torch.uint8) if case["fp8"] else s[c])[pages] for c in ("k_cache", "v_cache"))
        if case["fp8"]:
            k, v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
        for h in range(kv_heads):
            kh, vh = k[:, h].reshape(-1, dim)[:n].double(), v[:, h].reshape(-1, dim)[:n].double()
            if case["fp8"]:
                kh, vh = kh * s["k_scale"][h].double(), vh * s["v_scale"][h].double()
            group = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            out[i, group] = torch.softmax(s["q"][i, group].double() @ kh.T / math.sqrt(dim), -1) @ vh
    return out
