"""Rotary embedding with the append to a paged cache, and attention over it, against their definitions in 64 bits."""
import pytest
import torch

from tests import paged_util as P

pytestmark = pytest.mark.gpu


def _append(ops, qkv, heads, kv, dim, cos, sin, positions, table, cache, **kw):
    k, v, ks, vs = cache
    return ops.rope_append_paged(qkv, heads, kv, dim, cos, sin, positions, table, k, v, k_scale=ks, v_scale=vs, **kw)


@pytest.mark.parametrize("order", ["hnd", "nhd"])
@pytest.mark.parametrize("fp8", [False, True])
# one row; a decode batch; ragged prompts of sequences in any order; rows that share a CTA; rows of more vectors than a CTA has threads
@pytest.mark.parametrize("rows,heads,kv,dim,page", [(1, 32, 8, 128, 16), (37, 28, 4, 128, 24), (300, 4, 1, 64, 8), (5, 1, 1, 16, 1),
                                                    (3, 70, 5, 128, 32), (9, 8, 2, 256, 7)])
def test_append(rows, heads, kv, dim, page, fp8, order):
    from sharq_b200 import ops

    g = torch.Generator().manual_seed(rows + dim)
    seqs = max(1, rows // 3)
    # sequences of several rows, at scattered positions of their own
    per = torch.full((seqs,), rows // seqs)
    per[:rows % seqs] += 1
    reach = [int(n) + 11 + 3 * i for i, n in enumerate(per)]
    sequences = torch.cat([torch.full((int(n),), i) for i, n in enumerate(per)])
    positions = torch.cat([torch.randperm(r, generator=g)[:int(n)] for r, n in zip(reach, per)])
    mixed = torch.randperm(rows, generator=g)
    sequences, positions = (t[mixed].to(torch.int32).cuda() for t in (sequences, positions))
    table, pages = P.make_table(reach, page, 2, seed=rows)
    cache = P.make_cache(pages, kv, page, dim, fp8, 3, order)
    before = [c.clone() for c in cache[:2]]
    qkv = torch.randn(rows, (heads + 2 * kv) * dim + 24, generator=g).to(torch.bfloat16).cuda()[:, :(heads + 2 * kv) * dim + 8]
    cos, sin = P.rope_tables(max(reach), dim)
    q, k = _append(ops, qkv, heads, kv, dim, cos, sin, positions, table, cache, sequences=sequences, return_k=True)
    ops.check_device_errors()
    want_q, want_k, want_v = P.rotated64(qkv, heads, kv, dim, cos, sin, positions)
    # products of bf16 values are exact in float; the sum is rounded to float (2^-24) and to bf16 (2^-8)
    for got, want in ((q, want_q), (k, want_k)):
        assert bool(((got.double() - want).abs() <= 2.0 ** -8 * (1 + 2.0 ** -15) * want.abs()).all())
    pages_at = table[sequences.long(), (positions // page).long()].long()
    slots = (positions % page).long()
    for c, was, want, scale in zip(cache[:2], before, (want_k, want_v), cache[2:]):
        got = c[pages_at, :, slots]
        if fp8:
            # what a float division and one conversion give, to the bit; and within half a step (2^-4, or 2^-10 of the subnormal ones)
            exact = (want / scale.double()[:, None]).clamp(-448, 448)
            plain = (want.float() / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
            assert torch.equal(got.view(torch.uint8), plain.view(torch.uint8))
            assert bool(((got.double() - exact).abs() <= 2.0 ** -4 * (1 + 2.0 ** -15) * exact.abs() + 2.0 ** -10).all())
        else:
            assert bool(((got.double() - want).abs() <= 2.0 ** -8 * (1 + 2.0 ** -15) * want.abs()).all())
        # every other place is as it was
        was[pages_at, :, slots] = got
        assert torch.equal(c.contiguous().view(torch.uint8), was.contiguous().view(torch.uint8))
    # without the keys, and (one row per sequence) without a list of sequences
    only = _append(ops, qkv, heads, kv, dim, cos, sin, positions, table, cache, sequences=sequences)
    assert torch.equal(only, q)


@pytest.mark.parametrize("fp8", [False, True])
# rows whose threads take several heads, in numbers of heads that leave some without; heads that fill a CTA to the last thread
@pytest.mark.parametrize("rows,heads,kv,dim,page", [(700, 5, 1, 64, 8), (515, 70, 5, 128, 32), (512, 2, 1, 16, 1), (600, 13, 2, 80, 5),
                                                    (2, 510, 1, 80, 4), (513, 510, 1, 80, 4)])
def test_append_of_many_rows_or_heads(rows, heads, kv, dim, page, fp8):
    test_append(rows, heads, kv, dim, page, fp8, "hnd")


@pytest.mark.parametrize("fp8", [False, True])
def test_append_of_many_rows_equals_appends_of_few(fp8):
    from sharq_b200 import ops

    rows, heads, kv, dim, page = 1200, 7, 2, 64, 16
    g = torch.Generator().manual_seed(3)
    table, pages = P.make_table([600, 600], page, 2, 5)
    table[1, 20] = pages + 3  # no such page
    cos, sin = P.rope_tables(600, dim)
    qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g).to(torch.bfloat16).cuda()
    sequences = torch.arange(rows, dtype=torch.int32).cuda() % 2
    positions = torch.arange(rows, dtype=torch.int32).cuda() // 2
    positions[::13] = -1
    positions[70] = 600  # outside the tables
    a, b = (P.make_cache(pages, kv, page, dim, fp8, 3) for _ in range(2))
    qa, ka = _append(ops, qkv, heads, kv, dim, cos, sin, positions, table, a, sequences=sequences, return_k=True)
    parts = [_append(ops, qkv[i:i + 200], heads, kv, dim, cos, sin, positions[i:i + 200], table, b, sequences=sequences[i:i + 200], return_k=True)
             for i in range(0, rows, 200)]
    with pytest.raises(RuntimeError, match="cache"):
        ops.check_device_errors()
    for got, want in ((qa, torch.cat([p[0] for p in parts])), (ka, torch.cat([p[1] for p in parts])), (a[0], b[0]), (a[1], b[1])):
        assert torch.equal(got.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))
    assert bool(ka[70].isnan().all()) and not bool(ka[13].any())


def test_append_of_rows_without_sequences_equals_listed_ones():
    from sharq_b200 import ops

    table, pages = P.make_table([40, 3, 17], 16, 1, 5)
    cos, sin = P.rope_tables(64, 128)
    qkv = torch.randn(3, 48 * 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    positions = torch.tensor([39, 2, 16], dtype=torch.int32).cuda()
    a, b = (P.make_cache(pages, 8, 16, 128, False, 3) for _ in range(2))
    qa = _append(ops, qkv, 32, 8, 128, cos, sin, positions, table, a)
    qb = _append(ops, qkv, 32, 8, 128, cos, sin, positions, table, b, sequences=torch.arange(3, dtype=torch.int32).cuda())
    assert torch.equal(qa, qb) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_append_leaves_out_padding_and_reports_bad_places():
    from sharq_b200 import ops

    page, kv, dim, heads = 8, 2, 64, 4
    table, pages = P.make_table([16, 16, 16], page, 1, 5)
    table[2, 0] = pages  # one behind the last page
    cos, sin = P.rope_tables(64, dim)
    qkv = torch.randn(7, (heads + 2 * kv) * dim, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    #            padding, good, beyond the table of pages, bad page, bad sequences, beyond the tables of angles
    sequences = torch.tensor([0, 1, 1, 2, 3, -1, 0], dtype=torch.int32).cuda()
    positions = torch.tensor([-1, 15, 16, 3, 0, 0, 64], dtype=torch.int32).cuda()
    cache = P.make_cache(pages, kv, page, dim, False, 3)
    before = [c.clone() for c in cache[:2]]
    q, k = _append(ops, qkv, heads, kv, dim, cos, sin, positions, table, cache, sequences=sequences, return_k=True)
    with pytest.raises(RuntimeError, match="paged cache"):
        ops.check_device_errors()
    ops.check_device_errors()  # reported once
    assert bool((q[0] == 0).all()) and bool((k[0] == 0).all())
    assert bool(torch.isfinite(q[1]).all())
    assert bool(q[2:].isnan().all()) and bool(k[2:].isnan().all())
    for c, was in zip(cache[:2], before):
        was[table[1, 1], :, 7] = c[table[1, 1], :, 7]
        assert torch.equal(c, was)


SHAPES = [  # sequences' lengths, heads, kv_heads, dim, page size
    ([1], 32, 8, 128, 16),
    ([0], 4, 2, 128, 16),
    ([2, 0, 1, 63, 64, 65], 8, 8, 64, 16),
    ([97], 32, 8, 128, 16),
    ([15, 16, 17, 31, 32, 33, 0, 129], 28, 4, 128, 24),
    ([5000], 4, 1, 128, 64),
    ([777, 3, 2048, 1500], 16, 1, 128, 128),   # 16 query heads of one key/value head
    ([100, 900], 24, 1, 64, 7),                # 24: two pieces
    ([40, 41], 36, 2, 128, 1),                 # 18: two pieces, pages of one token
    ([300] * 40, 9, 3, 128, 32),               # many equal sequences
    ([3000, 1] + [0] * 5 + [64] * 70, 10, 2, 64, 256),
    ([20000, 5], 8, 8, 128, 64),               # parts of one (sequence, head) over many CTAs
    ([37 * i % 190 for i in range(331)], 8, 2, 128, 16),  # more sequences than a warp looks at at once
]


def wide(table, page):
    """The table with room for 200000 tokens per sequence: the form of attention goes by the room, not by the lengths."""
    out = torch.full((table.shape[0], 200000 // page), -1, dtype=torch.int32, device="cuda")
    out[:, :table.shape[1]] = table
    return out


@pytest.mark.parametrize("room", ["short", "wide"])
@pytest.mark.parametrize("order", ["hnd", "nhd"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lengths,heads,kv,dim,page", SHAPES)
def test_attention(lengths, heads, kv, dim, page, fp8, order, room):
    from sharq_b200 import ops

    table, pages = P.make_table(lengths, page, 2, seed=len(lengths))
    if room == "wide":
        table = wide(table, page)
    k, v, ks, vs = P.make_cache(pages, kv, page, dim, fp8, 7, order)
    g = torch.Generator().manual_seed(11)
    # rows of a merged activation: the heads of a row are contiguous, the rows are not
    merged = (2 * torch.randn(len(lengths), (heads + 2 * kv) * dim, generator=g)).to(torch.bfloat16).cuda()
    q = merged[:, :heads * dim].view(len(lengths), heads, dim)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    got = ops.paged_attention(q, k, v, table, n, k_scale=ks, v_scale=vs)
    ops.check_device_errors()
    out, size, reach = P.attention64(q, P.values64(k, ks), P.values64(v, vs), table, lengths)
    bound = P.attention_bound(out, size, reach, dim, max(lengths), fp8)
    assert bool(((got.double() - out).abs() <= bound).all()), float(((got.double() - out).abs() / bound).max())
    assert bool((got[torch.tensor(lengths) == 0] == 0).all())
    # the same bits again, into a given tensor
    again = torch.full_like(got, 7.0)
    assert ops.paged_attention(q, k, v, table, n, k_scale=ks, v_scale=vs, out=again) is not None
    assert torch.equal(again, got)


@pytest.mark.parametrize("room", ["short", "wide"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_ignores_what_lies_behind_a_sequence(dim, fp8, room):
    """NaN and infinities in slots behind the length and in pages of nobody, bad entries behind the last page."""
    from sharq_b200 import ops

    lengths, page = [5, 40, 0, 33], 16
    table, pages = P.make_table(lengths, page, 3, 1, unused=2 ** 30)
    k, v, ks, vs = P.make_cache(pages, 2, page, dim, fp8, 7)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for i, n in enumerate(lengths):
        for j in range(n):
            used[int(table[i, j // page]), j % page] = True
    used = used.cuda()
    if room == "wide":
        table = wide(table, page)
    q = torch.randn(4, 6, dim, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    clean = ops.paged_attention(q, k, v, table, n, k_scale=ks, v_scale=vs)
    for bad in (float("nan"), float("inf"), -float("inf")):
        dirty = [torch.where(used[:, None, :, None], c.float(), bad).to(c.dtype) for c in (k, v)]
        assert torch.equal(ops.paged_attention(q, *dirty, table, n, k_scale=ks, v_scale=vs), clean)
    ops.check_device_errors()


@pytest.mark.parametrize("room", ["short", "wide"])
def test_attention_reports_bad_lengths_and_pages(room):
    from sharq_b200 import ops

    page, dim = 16, 128
    for fp8 in (False, True):
        table, pages = P.make_table([64, 64, 64, 64, 64], page, 1, 1)
        if room == "wide":
            table = wide(table, page)
        k, v, ks, vs = P.make_cache(pages, 2, page, dim, fp8, 7)
        q = torch.randn(5, 8, dim, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
        good = ops.paged_attention(q, k, v, table, torch.full((5,), 64, dtype=torch.int32).cuda(), k_scale=ks, v_scale=vs)
        ops.check_device_errors()
        table[3, 2] = -1
        table[4, 3] = pages
        n = torch.tensor([64, -1, table.shape[1] * page + 1, 64, 64], dtype=torch.int32).cuda()
        got = ops.paged_attention(q, k, v, table, n, k_scale=ks, v_scale=vs)
        with pytest.raises(RuntimeError, match="paged cache"):
            ops.check_device_errors()
        assert torch.equal(got[0], good[0]) and bool(got[1:].isnan().all())
        n[4] = 48  # the bad page lies behind the last one in use
        got = ops.paged_attention(q, k, v, table, n, k_scale=ks, v_scale=vs)
        assert bool(torch.isfinite(got[4]).all())
        with pytest.raises(RuntimeError, match="paged cache"):
            ops.check_device_errors()


def test_attention_of_extreme_scores():
    """Scores far apart, equal, -inf through values of the cache, and a scale that is negative or zero."""
    from sharq_b200 import ops

    lengths, page, dim = [50, 200], 16, 128
    table, pages = P.make_table(lengths, page, 1, 1)
    for fp8 in (False, True):
        k, v, ks, vs = P.make_cache(pages, 1, page, dim, fp8, 7)
        q = (30 * torch.randn(2, 4, dim, generator=torch.Generator().manual_seed(2))).to(torch.bfloat16).cuda()
        q[1, 0] = 0
        q[1, 1] *= 2.0 ** -100
        n = torch.tensor(lengths, dtype=torch.int32).cuda()
        for scale in (None, 0.0, -0.5, 1.0):
            got = ops.paged_attention(q, k, v, table, n, scale=scale, k_scale=ks, v_scale=vs)
            out, size, reach = P.attention64(q, P.values64(k, ks), P.values64(v, vs), table, lengths, scale)
            bound = P.attention_bound(out, size, reach, dim, 200, fp8)
            assert bool(((got.double() - out).abs() <= bound).all()), (fp8, scale)
    # an infinite key: a score of -inf drops its token, one of +inf or NaN makes the row NaN
    k, v, _, _ = P.make_cache(pages, 1, page, dim, False, 7)
    at = (table[0, 0].item(), 0, 3)
    k[at][0] = float("inf")
    q = q.abs()
    q[0, 1, 0] = -1
    got = ops.paged_attention(q, k, v, table, n)
    out, size, reach = P.attention64(q, P.values64(k, None), P.values64(v, None), table, lengths)
    assert bool(got[0, 0].isnan().all()) and bool(torch.isfinite(got[0, 1]).all())
    k[at][0] = 0
    k[at][1:] = -30000  # in its place a score that is as good as -inf: its probability is 0 either way
    q[0, 1, 0] = 1
    lo = ops.paged_attention(q, k, v, table, n)[0, 1]
    out, size, reach = P.attention64(q, P.values64(k, None), P.values64(v, None), table, lengths)
    assert bool(((lo.double() - out[0, 1]).abs() <= P.attention_bound(out, size, reach, dim, 200, False)[0, 1]).all())


def test_attention_far_into_a_large_cache():
    """Offsets beyond 2^31 elements and 2^32 bytes."""
    from sharq_b200 import ops

    kv, page, dim = 8, 128, 128
    pages = 2 ** 32 // (kv * page * dim * 2) + 3
    k = torch.zeros(pages, kv, page, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    last = pages - 1
    g = torch.Generator().manual_seed(2)
    cos, sin = P.rope_tables(256, dim)
    table = torch.tensor([[last, last - 1]], dtype=torch.int32).cuda()
    qkv = torch.randn(200, (16 + 2 * kv) * dim, generator=g).to(torch.bfloat16).cuda()
    positions = torch.arange(200, dtype=torch.int32).cuda()
    q = ops.rope_append_paged(qkv, 16, kv, dim, cos, sin, positions, table, k, v, sequences=torch.zeros(200, dtype=torch.int32).cuda())
    got = ops.paged_attention(q[-1:], k, v, table, torch.tensor([200], dtype=torch.int32).cuda())
    ops.check_device_errors()
    assert not bool(k[:last - 1].any())
    small = torch.tensor([[0, 1]], dtype=torch.int32).cuda()
    want, size, reach = P.attention64(q[-1:], *(P.values64(c[[last, last - 1]], None) for c in (k, v)), small, [200])
    assert bool(((got.double() - want).abs() <= P.attention_bound(want, size, reach, dim, 200, False)).all())


def test_refusals():
    from sharq_b200 import ops

    table, pages = P.make_table([40, 30], 16, 1, 5)
    k, v, _, _ = P.make_cache(pages, 2, 16, 128, False, 3)
    k8, v8, ks, vs = P.make_cache(pages, 2, 16, 128, True, 3)
    cos, sin = P.rope_tables(64, 128)
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16).cuda()
    n = torch.tensor([1, 2], dtype=torch.int32).cuda()
    qkv = torch.zeros(2, 8 * 128, dtype=torch.bfloat16).cuda()

    def attend(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            ops.paged_attention(*args, **kw)

    attend("CUDA bfloat16", q.float(), k, v, table, n)
    attend("multiple of the cache's heads", q[:, :3], k, v, table, n)
    attend("head_dim", q[..., :64].contiguous(), k, v, table, n)
    attend("heads are contiguous", q.transpose(1, 2), k, v, table, n)
    attend("k_scale", q, k8, v8, table, n)
    attend("k_scale", q, k, v, table, n, k_scale=ks, v_scale=vs)
    attend("k_scale", q, k8, v8, table, n, k_scale=ks[:1], v_scale=vs)
    attend("alike", q, k, v8, table, n)
    attend("alike", q, k, v[1:], table, n)
    attend("bfloat16 or torch.float8_e4m3fn", q, k.half(), v.half(), table, n)
    attend("overlap", q, k[:1].expand(pages, -1, -1, -1), v[:1].expand(pages, -1, -1, -1), table, n)
    attend("int32", q, k, v, table.long(), n)
    attend("int32", q, k, v, table, n.long())
    attend("row for every row", q, k, v, table[:1], n)
    attend("page_table must not be empty", q, k, v, table[:, :0], n)
    attend("out must be", q, k, v, table, n, out=torch.empty_like(q).float())
    attend("head_dim must be 64 or 128", q[..., :32].contiguous(), k[..., :32].contiguous(), v[..., :32].contiguous(), table, n)
    attend("multiples of 8", torch.zeros(2, 4 * 128 + 4, dtype=torch.bfloat16).cuda()[:, 4:].view(2, 4, 128), k, v, table, n)

    def append(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            ops.rope_append_paged(*args, **kw)

    append("unit column stride", qkv.t(), 4, 2, 128, cos, sin, n, table, k, v)
    append("exceeds the row width", qkv[:, :-8], 4, 2, 128, cos, sin, n, table, k, v)
    append("cos must be", qkv, 4, 2, 128, cos.float(), sin, n, table, k, v)
    append("sin must be", qkv, 4, 2, 128, cos, sin[:-1], n, table, k, v)
    append("positions must be", qkv, 4, 2, 128, cos, sin, n.long(), table, k, v)
    append("sequences must be", qkv, 4, 2, 128, cos, sin, n, table, k, v, sequences=n[:1])
    append("row for every row", qkv, 4, 2, 128, cos, sin, n, table[:1], k, v)
    append("kv_heads heads", qkv, 6, 1, 128, cos, sin, n, table, k, v)
    append("16-byte aligned", torch.zeros(2, 8 * 128 + 8, dtype=torch.bfloat16).cuda()[:, 4:], 4, 2, 128, cos, sin, n, table, k, v)
    # nothing to do
    assert ops.paged_attention(q[:0], k, v, table, n[:0]).shape == (0, 4, 128)
    assert ops.rope_append_paged(qkv[:0], 4, 2, 128, cos, sin, n[:0], table, k, v).shape == (0, 4, 128)


def test_append_divides_as_a_float_division():
    """Every finite bf16 value, infinities and NaN, by scales of many sizes, in a cache of e4m3 values: the bits of a float division, clamped
    and converted (a NaN's sign aside)."""
    from sharq_b200 import ops

    dim = 128
    values = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(512, dim)
    g = torch.Generator().manual_seed(4)
    scales = torch.cat((torch.rand(40, generator=g) * 0.1 + 1e-4, 2.0 ** torch.arange(-20, 20, 8).float(), torch.tensor([1.9999999, 3e-33, 1e-39, 7e35])))
    kv = scales.numel()
    qkv = torch.zeros(512, (1 + 2 * kv) * dim, dtype=torch.bfloat16)
    qkv[:, (1 + kv) * dim:] = values.repeat(1, kv)
    table, pages = P.make_table([512], 16, 0, 1)
    k, v = (torch.zeros(pages, kv, 16, dim, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    cos, sin = P.rope_tables(512, dim)
    at = torch.arange(512, dtype=torch.int32).cuda()
    ops.rope_append_paged(qkv.cuda(), 1, kv, dim, cos, sin, at, table, k, v, sequences=torch.zeros_like(at), k_scale=scales.cuda(),
                          v_scale=scales.cuda())
    ops.check_device_errors()
    got = v[table[0].long()].transpose(1, 2).reshape(512, kv, dim)
    want = (values.cuda().float()[:, None] / scales.cuda()[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    nan = want.float().isnan()
    assert torch.equal(got.float().isnan(), nan)
    assert torch.equal(got.view(torch.uint8)[~nan], want.view(torch.uint8)[~nan])


def _attention_inputs(seed, lengths, heads=8, kv=2, dim=128, page=16, fp8=False, room="wide"):
    table, pages = P.make_table(lengths, page, 1, seed)
    k, v, ks, vs = P.make_cache(pages, kv, page, dim, fp8, seed)
    q = torch.randn(len(lengths), heads, dim, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    return (q, k, v, wide(table, page) if room == "wide" else table, n), dict(k_scale=ks, v_scale=vs)


@pytest.mark.parametrize("room", ["short", "wide"])
def test_attention_on_two_streams_and_in_two_graphs(room):
    """Calls that overlap have scratch of their own; a replay reads the lengths that are there then."""
    from sharq_b200 import ops

    calls = [_attention_inputs(1, [3000, 17, 400], room=room), _attention_inputs(2, [2500, 1, 0, 90], fp8=True, room=room)]
    want = [ops.paged_attention(*a, **kw) for a, kw in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    outs = [[torch.empty_like(w) for _ in range(30)] for w in want]
    for i in range(30):
        for s, (a, kw), o in zip(streams, calls, outs):
            with torch.cuda.stream(s):
                ops.paged_attention(*a, **kw, out=o[i])
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)
    graphs = []
    for a, kw in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.paged_attention(*a, **kw)
        graphs.append((g, out))
    for _ in range(5):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, (_, out) in zip(want, graphs):
        assert torch.equal(w, out)
    (q, k, v, table, n), kw = calls[0]
    n.copy_(torch.tensor([5, 0, 399], dtype=torch.int32))
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], ops.paged_attention(q, k, v, table, n, **kw))
    ops.check_device_errors()


def test_attention_of_shared_pages_drafts_and_broadcast_queries():
    """A sequence in several rows with lengths of its own, pages that sequences share, queries of one head for all, into its own queries."""
    from sharq_b200 import ops

    (q, k, v, table, n), kw = _attention_inputs(3, [300, 40], room="short")
    rows = torch.tensor([0, 0, 0, 1]).cuda()
    lengths = [298, 299, 300, 40]
    table4 = table[rows].contiguous()
    table4[3, 0] = table4[0, 0]  # a shared prefix
    one = q[:1, :1].expand(4, 8, 128)
    got = ops.paged_attention(one, k, v, table4, torch.tensor(lengths, dtype=torch.int32).cuda())
    out, size, reach = P.attention64(one, P.values64(k, None), P.values64(v, None), table4, lengths)
    assert bool(((got.double() - out).abs() <= P.attention_bound(out, size, reach, 128, 300, False)).all())
    want = ops.paged_attention(q, k, v, table, n)
    assert ops.paged_attention(q, k, v, table, n, out=q) is not None
    assert torch.equal(q, want)
    ops.check_device_errors()


@pytest.mark.parametrize("room", ["short", "wide"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_with_infinite_and_with_the_largest_values(dim, room):
    """An infinite value of a token that counts is infinite in the result, whatever its probability; the mean of finite ones is finite."""
    from sharq_b200 import ops

    lengths, page, kv = [1, 40, 700, 5000], 16, 2
    table, pages = P.make_table(lengths, page, 1, 1)
    k, v, _, _ = P.make_cache(pages, kv, page, dim, False, 7)
    largest = torch.finfo(torch.bfloat16).max
    v[..., 5] = float("inf")
    v[..., 6] = -float("inf")
    v[..., 7] = largest
    v[..., 8] = -largest
    for i, n in enumerate(lengths):  # one token of every sequence
        v[table[i, (n // 2) // page].long(), :, n // 2 % page, 9] = float("inf")
    if room == "wide":
        table = wide(table, page)
    q = torch.randn(4, 6, dim, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    got = ops.paged_attention(q, k, v, table, n)
    ops.check_device_errors()
    assert bool((got[..., [5, 9]] == float("inf")).all()) and bool((got[..., 6] == -float("inf")).all())
    # the mean is the largest value but for roundings of some 2^-23 of it, which bf16 does not see
    assert bool((got[..., 7] == largest).all()) and bool((got[..., 8] == -largest).all())
    rest = [d for d in range(dim) if d not in (5, 6, 7, 8, 9)]
    out, size, reach = P.attention64(q, P.values64(k, None), P.values64(v, None), table, lengths)
    bound = P.attention_bound(out, size, reach, dim, max(lengths), False)
    assert bool(((got.double() - out).abs() <= bound)[..., rest].all())


def test_a_length_near_the_end_of_an_int_is_reported():
    from sharq_b200 import ops

    page = 65536
    k, v = (torch.zeros(1, 1, page, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.zeros(2, 32768, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    n = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, k, v, table, n)
    with pytest.raises(RuntimeError, match="paged cache"):
        ops.check_device_errors()
    assert bool(got.isnan().all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim,group", [(64, 3), (128, 12), (128, 1), (64, 16)])
def test_attention_of_few_sequences_at_every_size_of_cluster(dim, group, fp8):
    """Tables of one to some hundred tiles, with sequences that leave warps and CTAs of their cluster without a token."""
    from sharq_b200 import ops

    page, kv = 16, 2
    for longest in (1, 16, 17, 33, 128, 129, 255, 257, 400, 513, 1000, 1025, 2049, 3000):
        for lengths in ([longest], [longest, 0, 1, longest // 2 + 1, longest // 3]):
            table, pages = P.make_table(lengths, page, 1, seed=longest)
            k, v, ks, vs = P.make_cache(pages, kv, page, dim, fp8, longest)
            g = torch.Generator().manual_seed(longest)
            q = torch.randn(len(lengths), kv * group, dim, generator=g).to(torch.bfloat16).cuda()
            n = torch.tensor(lengths, dtype=torch.int32).cuda()
            got = ops.paged_attention(q, k, v, table, n, k_scale=ks, v_scale=vs)
            out, size, reach = P.attention64(q, P.values64(k, ks), P.values64(v, vs), table, lengths)
            bound = P.attention_bound(out, size, reach, dim, longest, fp8)
            assert bool(((got.double() - out).abs() <= bound).all()), (longest, lengths)
    ops.check_device_errors()


@pytest.mark.parametrize("fp8", [False, True])
# clusters of one CTA in numbers that fill two, three and more CTAs per SM, and more than the direct form takes
@pytest.mark.parametrize("seqs,heads,kv,dim,longest", [(37, 32, 8, 128, 300), (38, 32, 8, 128, 300), (55, 8, 8, 64, 200), (111, 12, 4, 128, 500),
                                                       (56, 32, 8, 64, 100), (74, 32, 8, 128, 90), (75, 32, 8, 128, 90), (45, 72, 8, 128, 150)])
def test_attention_of_many_short_sequences(seqs, heads, kv, dim, longest, fp8):
    from sharq_b200 import ops

    lengths = [(i * 37) % (longest + 1) for i in range(seqs - 1)] + [longest]
    page = 16
    table, pages = P.make_table(lengths, page, 1, seed=seqs)
    k, v, ks, vs = P.make_cache(pages, kv, page, dim, fp8, 5)
    q = torch.randn(seqs, heads, dim, generator=torch.Generator().manual_seed(seqs)).to(torch.bfloat16).cuda()
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    got = ops.paged_attention(q, k, v, table, n, k_scale=ks, v_scale=vs)
    ops.check_device_errors()
    out, size, reach = P.attention64(q, P.values64(k, ks), P.values64(v, vs), table, lengths)
    bound = P.attention_bound(out, size, reach, dim, longest, fp8)
    assert bool(((got.double() - out).abs() <= bound).all()), float(((got.double() - out).abs() / bound).max())
    assert torch.equal(ops.paged_attention(q, k, v, table, n, k_scale=ks, v_scale=vs), got)


@pytest.mark.parametrize("kv,group,lengths", [(40000, 1, [65]), (33000, 1, [33, 1, 97]), (3000, 20, [70])])
def test_attention_of_very_many_heads(kv, group, lengths):
    """Items whose tiles fall to several warps at every index of a head, and of a piece of a group, that the interface takes."""
    from sharq_b200 import ops

    page, dim = 16, 64
    table, pages = P.make_table(lengths, page, 1, seed=3)
    g = torch.Generator(device="cuda").manual_seed(7)
    k, v = (torch.randn(pages, kv, page, dim, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q = torch.randn(len(lengths), kv * group, dim, generator=g, device="cuda", dtype=torch.bfloat16)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    got = torch.full_like(q, 7.0)
    ops.paged_attention(q, k, v, table, n, out=got)
    ops.check_device_errors()
    out, size, reach = P.attention64(q, P.values64(k, None), P.values64(v, None), table, lengths)
    bound = P.attention_bound(out, size, reach, dim, max(lengths), False)
    assert bool(((got.double() - out).abs() <= bound).all()), float(((got.double() - out).abs() / bound).max())


@pytest.mark.parametrize("room", ["short", "wide"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dim,group", [(64, 3), (128, 4), (128, 12)])
def test_attention_of_values_that_nearly_cancel(dim, group, fp8, room):
    """Values of +-448 under probabilities that differ by a few thousandths: 11 bits of a probability are too few for the difference, with
    a cache of either type.  (16 bits, as attention_bound has them for bf16.)"""
    from sharq_b200 import ops

    lengths, page, kv = [2, 34, 4, 1], 16, 2
    table, pages = P.make_table(lengths, page, 1, seed=4)
    g = torch.Generator().manual_seed(group)
    k = torch.randn(pages, kv, page, dim, generator=g).to(torch.float8_e4m3fn)
    sign = 1 - 2 * (torch.arange(page) % 2)
    v = (448.0 * sign[None, None, :, None]).expand(pages, kv, page, dim).to(torch.float8_e4m3fn).contiguous()
    k, v = (x.cuda() if fp8 else x.float().to(torch.bfloat16).cuda() for x in (k, v))
    ks, vs = (torch.tensor([1.0, 0.25], device="cuda"), torch.tensor([0.5, 1.0], device="cuda")) if fp8 else (None, None)
    q = (2.0 ** -7 * torch.randn(len(lengths), kv * group, dim, generator=g)).to(torch.bfloat16).cuda()
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    got = ops.paged_attention(q, k, v, wide(table, page) if room == "wide" else table, n, k_scale=ks, v_scale=vs)
    ops.check_device_errors()
    out, size, reach = P.attention64(q, P.values64(k, ks), P.values64(v, vs), table, lengths)
    bound = P.attention_bound(out, size, reach, dim, max(lengths), False)
    assert bool(((got.double() - out).abs() <= bound).all()), float(((got.double() - out).abs() / bound).max())
