"""Paged caches for tests, and the cache operators from their definitions in 64 bits."""
import math

import torch


def make_cache(pages, kv_heads, page_size, dim, fp8, seed, order="hnd", device="cuda"):
    """(k, v, k_scale, v_scale): a cache with values everywhere; order "nhd" puts the tokens of a page before its heads."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        shape = (pages, kv_heads, page_size, dim) if order == "hnd" else (pages, page_size, kv_heads, dim)
        x = 1.5 * torch.randn(shape, generator=g)
        x[..., 3] *= 4
        x = (x / 0.03).clamp(-448, 448).to(torch.float8_e4m3fn) if fp8 else x.to(torch.bfloat16)
        x = x.to(device)
        out.append(x if order == "hnd" else x.transpose(1, 2))
    if not fp8:
        return (*out, None, None)
    scales = [(0.02 + 0.02 * torch.rand(kv_heads, generator=g)).to(device) for _ in range(2)]
    return (*out, *scales)


def make_table(lengths, page_size, spare, seed, unused=-1, device="cuda"):
    """(page table int32 [sequences, most pages], pages of the cache): scattered pages, `unused` behind the last of a sequence."""
    counts = [-(-n // page_size) for n in lengths]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), max(1, max(counts, default=1))), unused, dtype=torch.int32)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table.to(device), pages


def values64(cache, scale):
    """What the cache stands for, float64 [pages, kv_heads, page_size, dim]."""
    x = cache.float().double()
    return x if scale is None else x * scale.double()[:, None, None]


def attention64(q, k, v, table, lengths, scale=None):
    """-> (out, sum_j p_j |v_j|, largest sum_d |q_d k_jd| * scale) in float64; k, v from values64."""
    seqs, heads, dim = q.shape
    kv_heads, page = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros(seqs, heads, dim, dtype=torch.float64, device=q.device)
    size, reach = torch.zeros_like(out), torch.zeros(seqs, heads, 1, dtype=torch.float64, device=q.device)
    for i, n in enumerate(lengths):
        if n <= 0:
            continue
        pages = table[i, :-(-n // page)].long()
        ki, vi = (x[pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :n] for x in (k, v))
        qi = q[i].double().view(kv_heads, heads // kv_heads, dim)
        p = torch.softmax(qi @ ki.transpose(1, 2) * scale, -1)
        out[i] = (p @ vi).view(heads, dim)
        size[i] = (p @ vi.abs()).view(heads, dim)
        reach[i] = (qi.abs() @ ki.abs().transpose(1, 2) * abs(scale)).amax(-1).view(heads, 1)
    return out, size, reach


def attention_bound(out, size, reach, dim, longest, fp8):
    """How far the kernel may be from attention64, element by element.
    A score is a float sum of dim exact products: off by at most (dim + 4) * 2^-23 of the sum of their sizes (`reach`), the multiplication by
    the scale and the exponential's argument among the 4; a probability is off by that, relative, twice (its own and its sum's).  It is
    rounded to two bf16 numbers (2^-16) or to f16 (2^-11) for the product, and the product's float sum has at most longest + 16 roundings of 2^-23 and the
    joins.  All that in units of sum p |v|; the result is rounded to bf16 once (2^-8)."""
    score = (dim + 4) * 2.0 ** -23 * reach
    rounding = 2.0 ** -11 if fp8 else 2.0 ** -16
    return (rounding + 2 * score * (1 + score) + 2 * (longest + 64) * 2.0 ** -23) * size + 2.0 ** -8 * (1 + 2.0 ** -7) * out.abs() + 1e-30


def rotated64(qkv, heads, kv_heads, dim, cos, sin, positions):
    """(q, k, v) [rows, heads, dim] in float64, positions clamped into the tables."""
    rows = qkv.shape[0]
    x = qkv[:, :(heads + 2 * kv_heads) * dim].double().reshape(rows, -1, dim)
    at = positions.long().clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]
    qk = x[:, :heads + kv_heads]
    qk = qk * c + torch.cat((-qk[..., dim // 2:], qk[..., :dim // 2]), -1) * s
    return qk[:, :heads], qk[:, heads:], x[:, heads + kv_heads:]


def rope_tables(n, dim, device="cuda"):
    ang = torch.outer(torch.arange(n, dtype=torch.float64), 5e5 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim))
    ang = torch.cat((ang, ang), -1)
    return ang.cos().to(torch.bfloat16).to(device), ang.sin().to(torch.bfloat16).to(device)
