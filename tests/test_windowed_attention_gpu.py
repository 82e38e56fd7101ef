"""Attention of single tokens over a paged cache with a sliding window and first tokens that stay visible (ops.paged_attention)."""
import math

import pytest
import torch

from sharq_b200 import ops
from tests.paged_util import attention_bound, make_cache, make_table, values64

pytestmark = pytest.mark.gpu


def seen_of(n, window, sinks):
    return [j for j in range(n) if j < sinks or n - 1 - j < window]


def definition64(q, k, v, table, lengths, window, sinks, scale):
    """attention_bound's arguments: (out, sum_j p_j |v_j|, largest sum_d |q_d k_jd| * scale) over the tokens that are seen, and no others."""
    seqs, heads, dim = q.shape
    kv_heads, page = k.shape[1], k.shape[2]
    out = torch.zeros(seqs, heads, dim, dtype=torch.float64, device=q.device)
    size, reach = torch.zeros_like(out), torch.zeros(seqs, heads, 1, dtype=torch.float64, device=q.device)
    for i, n in enumerate(lengths):
        if n <= 0:
            continue
        j = torch.tensor(seen_of(n, window, sinks), device=q.device)
        pages = table[i].long()[j // page]
        ki, vi = (x[pages, :, j % page].transpose(0, 1) for x in (k, v))
        qi = q[i].double().view(kv_heads, heads // kv_heads, dim)
        p = torch.softmax(qi @ ki.transpose(1, 2) * scale, -1)
        out[i], size[i] = (p @ vi).view(heads, dim), (p @ vi.abs()).view(heads, dim)
        reach[i] = (qi.abs() @ ki.abs().transpose(1, 2) * abs(scale)).amax(-1).view(heads, 1)
    return out, size, reach


def run(lengths, heads, kv_heads, dim, page, fp8, window, sinks, seed=1, order="hnd", wide=0, scale=None):
    """The operator against the definition; everything that no sequence sees is NaN, and its pages are no pages."""
    table, pages = make_table(lengths, page, 2, seed)
    k, v, k_scale, v_scale = make_cache(pages, kv_heads, page, dim, fp8, seed, order)
    seen = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    rows = table.tolist()
    for i, n in enumerate(lengths):
        used = seen_of(n, window, sinks)
        for j in used:
            seen[rows[i][j // page], j % page] = True
        alive = {j // page for j in used}
        for at in range(len(rows[i])):
            if at not in alive:
                table[i, at] = (-1, 10 ** 9, pages)[at % 3]
    hidden = ~seen[:, None].expand(pages, kv_heads, page)
    for x in (k, v):
        x.view(torch.uint8)[hidden] = 0x7F if fp8 else 0xFF  # NaN
    if wide:
        table = torch.cat((table, torch.full((len(lengths), wide), -1, dtype=torch.int32, device="cuda")), 1)
    q = torch.randn(len(lengths), heads, dim, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
    at = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, k, v, table, at, scale=scale, k_scale=k_scale, v_scale=v_scale, window=window, sinks=sinks)
    want, size, reach = definition64(q, values64(k, k_scale), values64(v, v_scale), table, lengths, window, sinks, dim ** -0.5 if scale is None else scale)
    limit = attention_bound(want, size, reach, dim, window + sinks, fp8)
    assert ((got.double() - want).abs() <= limit).all()
    ops.check_device_errors()
    return got


WINDOWS = [(1, 0), (1, 1), (16, 0), (33, 4), (100, 5), (128, 64), (500, 33), (4000, 4)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (7, 1, 128, 24), (32, 2, 64, 64), (4, 4, 64, 7), (40, 2, 128, 8)])
def test_mixed_lengths(fp8, window, sinks, heads, kv_heads, dim, page):
    run([1, 700, 0, 33, 34, 160, 1023, 17, 5, 2000], heads, kv_heads, dim, page, fp8, window, sinks)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 129, 1000, 4097])
def test_one_sequence(fp8, length):
    for window, sinks in ((1, 0), (16, 16), (32, 3), (64, 0), (65, 20)):
        run([length], 8, 2, 128, 16, fp8, window, sinks, seed=length)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window,sinks", [(40, 4), (1000, 100), (6000, 0)])
def test_many_sequences_and_wide_tables(fp8, window, sinks):
    """So many that their tiles are one list, and tables as wide as a cache of longer sequences has."""
    g = torch.Generator().manual_seed(window)
    lengths = (torch.rand(150, generator=g) ** 2 * 3000).int().tolist()
    run(lengths, 8, 4, 64, 32, fp8, window, sinks, wide=500)
    run([9000, 0, 20011, 5], 4, 1, 128, 128, fp8, window, sinks, wide=100)


@pytest.mark.parametrize("order", ["hnd", "nhd"])
@pytest.mark.parametrize("scale", [None, -0.3, 1.0])
def test_orders_and_scales(order, scale):
    run([300, 77, 1200], 8, 2, 64, 16, False, 130, 6, order=order, scale=scale)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_window_of_everything_is_no_window(fp8):
    lengths = [1, 400, 0, 31, 2100]
    table, pages = make_table(lengths, 16, 2, 3)
    k, v, k_scale, v_scale = make_cache(pages, 2, 16, 128, fp8, 3)
    q = torch.randn(5, 8, 128, device="cuda").to(torch.bfloat16)
    at = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = ops.paged_attention(q, k, v, table, at, k_scale=k_scale, v_scale=v_scale)
    for window, sinks in ((2100, 0), (10 ** 12, 4), (2000, 100), (1, 2100), (1, 10 ** 12)):
        got = ops.paged_attention(q, k, v, table, at, k_scale=k_scale, v_scale=v_scale, window=window, sinks=sinks)
        assert torch.equal(got, want)
    assert torch.equal(want, ops.paged_attention(q, k, v, table, at, k_scale=k_scale, v_scale=v_scale, window=None, sinks=7))
    ops.check_device_errors()


def test_bad_pages_and_lengths_are_reported():
    lengths = [500, 40, 200]
    for window, bad in ((100, 499), (100, 401), (100, 3)):
        table, pages = make_table(lengths, 16, 2, 4)
        k, v, *_ = make_cache(pages, 2, 16, 64, False, 4)
        q = torch.randn(3, 4, 64, device="cuda").to(torch.bfloat16)
        at = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        want = ops.paged_attention(q, k, v, table, at, window=window, sinks=4)
        table[0, bad // 16] = pages
        got = ops.paged_attention(q, k, v, table, at, window=window, sinks=4)
        assert got[0].isnan().all() and torch.equal(got[1:], want[1:])
        with pytest.raises(RuntimeError, match="paged cache"):
            ops.check_device_errors()
    at[1] = table.shape[1] * 16 + 1
    assert ops.paged_attention(q, k, v, table, at, window=window, sinks=4)[1].isnan().all()
    with pytest.raises(RuntimeError, match="paged cache"):
        ops.check_device_errors()


def test_captured():
    lengths = [300, 900]
    table, pages = make_table([1000, 1000], 16, 2, 5)
    k, v, *_ = make_cache(pages, 2, 16, 128, False, 5)
    q = torch.randn(2, 8, 128, device="cuda").to(torch.bfloat16)
    at = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ops.paged_attention(q, k, v, table, at, window=64, sinks=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.paged_attention(q, k, v, table, at, window=64, sinks=4)
    for _ in range(3):
        at += 37
        graph.replay()
        want = ops.paged_attention(q, k, v, table, at, window=64, sinks=4)
        torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
    # the last step takes the second sequence beyond what its row of the table holds
    assert got[0].isfinite().all() and got[1].isnan().all()
    with pytest.raises(RuntimeError, match="paged cache"):
        ops.check_device_errors()


def test_refusals():
    table, pages = make_table([30], 16, 2, 1)
    k, v, *_ = make_cache(pages, 2, 16, 64, False, 1)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([30], dtype=torch.int32, device="cuda")
    for window, sinks in ((0, 0), (-1, 0), (5, -1), (None, -1)):
        with pytest.raises(RuntimeError, match="window|sinks"):
            ops.paged_attention(q, k, v, table, at, window=window, sinks=sinks)
    assert math.isfinite(float(ops.paged_attention(q, k, v, table, at, window=5).float().sum()))
