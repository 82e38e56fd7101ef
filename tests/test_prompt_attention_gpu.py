"""Attention of ragged prompts (ops.prompt_attention) against its definition in 64 bits."""
import math

import pytest
import torch

from sharq_b200 import ops

pytestmark = pytest.mark.gpu


def definition64(q, k, v, lengths, key_lengths, window, sinks, scale):
    """-> (out, sum_j p_j |v_j|, largest sum_d |q_d k_jd| * scale) in float64, row by row over the keys that it sees and no others."""
    rows, heads, dim = q.shape
    kv_heads = k.shape[1]
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device=q.device)
    size, reach = torch.zeros_like(out), torch.zeros(rows, heads, 1, dtype=torch.float64, device=q.device)
    q0 = k0 = 0
    for n, m in zip(lengths, key_lengths):
        p = torch.arange(m - n, m, device=q.device)[:, None]
        j = torch.arange(m, device=q.device)
        seen = (j <= p) & ((p - j < window) | (j < sinks)) if window else j <= p
        for h in range(kv_heads if m else 0):
            group = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            qh = q[q0:q0 + n, group].double().transpose(0, 1)
            kh, vh = (x[k0:k0 + m, h].double() for x in (k, v))
            a = torch.where(seen, qh @ kh.T * scale, -math.inf)
            w = torch.softmax(a, -1)
            w = torch.where(seen.any(-1)[:, None], w, 0)
            bad = ~vh.isfinite().all(-1)
            if bad.any():  # such a value reaches the rows that see it, and no others
                w0 = torch.where(bad, 0, w) @ torch.where(bad[:, None], 0, vh)
                for i in bad.nonzero()[:, 0].tolist():
                    w0 = torch.where(seen[:, i, None], w0 + w[..., i, None] * vh[i], w0)
                out[q0:q0 + n, group] = w0.transpose(0, 1)
            else:
                out[q0:q0 + n, group] = (w @ vh).transpose(0, 1)
            size[q0:q0 + n, group] = (w @ vh.abs().nan_to_num(0.0, 0.0)).transpose(0, 1)
            far = torch.where(seen, qh.abs() @ kh.abs().T * abs(scale), 0).amax(-1)
            reach[q0:q0 + n, group] = far.T[..., None]
        q0, k0 = q0 + n, k0 + m
    return out, size, reach


def bound(out, size, reach, dim, longest):
    """How far the kernel may be from the definition, element by element.
    A score is a float sum of dim exact products: off by at most (dim + 4) * 2^-23 of the sum of their sizes, the multiplication by the scale and
    the exponential's argument among the 4; a probability is off by that, relative, twice (its own and its sum's), and by 2^-18 for the exponent's shift
    by 32, whose float step is 2^-19.  It is rounded to bf16 (2^-8); the product's float sum has at most longest + 64 roundings of 2^-23.  All that in units of sum p |v|; the
    result is rounded to bf16 once (2^-8)."""
    score = (dim + 4) * 2.0 ** -23 * reach + 2.0 ** -18
    return (2.0 ** -8 + 2 * score * (1 + score) + 2 * (longest + 64) * 2.0 ** -23) * size + 2.0 ** -8 * (1 + 2.0 ** -7) * out.abs() + 1e-30


def ends(lengths):
    return torch.tensor([0, *torch.tensor(lengths, dtype=torch.int64).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def inputs(lengths, key_lengths, heads, kv_heads, dim, seed, behind=0):
    """Values are the last columns of a wider activation; `behind` rows of no sequence, which hold NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, keys = sum(lengths), sum(key_lengths)
    rand = lambda n, w: torch.randn(n, w, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    q, k, v = rand(rows + behind, heads * dim), rand(keys + behind, kv_heads * dim), rand(keys + behind, (heads + kv_heads) * dim)
    q[:, ::29] *= 3
    k[:, ::31] *= 2
    q[rows:], k[keys:], v[keys:] = math.nan, math.nan, math.nan
    return q.view(-1, heads, dim), k.view(-1, kv_heads, dim), v[:, heads * dim:].view(-1, kv_heads, dim)


def check(got, q, k, v, lengths, key_lengths, window=None, sinks=0, scale=None):
    rows, dim = sum(lengths), q.shape[2]
    want, size, reach = definition64(q[:rows], k, v, lengths, key_lengths, window or 0, sinks if window else 0, dim ** -0.5 if scale is None else scale)
    limit = bound(want, size, reach, dim, max(key_lengths, default=0))
    got = got[:rows].double()
    fine = want.isfinite()
    assert torch.equal(fine, got.isfinite()) and torch.equal(want.isnan(), got.isnan())
    assert torch.equal(want[~fine & ~want.isnan()], got[~fine & ~want.isnan()])
    over = ((got - want).abs() > limit) & fine
    assert not over.any(), (over.nonzero()[:5].tolist(), got[over][:5].tolist(), want[over][:5].tolist())


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (7, 1, 128), (3, 3, 64), (4, 4, 128), (16, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (1, 1), (5, 3), (64, 4), (128, 0), (200, 9), (130, 300), (10 ** 6, 4)])
def test_ragged_prompts(heads, kv_heads, dim, window, sinks):
    lengths = [1, 0, 257, 2, 700, 31, 128, 64, 0]
    q, k, v = inputs(lengths, lengths, heads, kv_heads, dim, heads + sinks)
    got = ops.prompt_attention(q, k, v, ends(lengths), window=window, sinks=sinks)
    check(got, q, k, v, lengths, lengths, window, sinks)
    ops.check_device_errors()
    assert torch.equal(got, ops.prompt_attention(q, k, v, ends(lengths), window=window, sinks=sinks))


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 1000, 3000])
@pytest.mark.parametrize("dim,window,sinks", [(128, None, 0), (64, 100, 4), (128, 100, 4), (128, 1000, 130)])
def test_lengths(length, dim, window, sinks):
    q, k, v = inputs([length], [length], 4, 2, dim, length)
    check(ops.prompt_attention(q, k, v, ends([length]), window=window, sinks=sinks), q, k, v, [length], [length], window, sinks)
    ops.check_device_errors()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 0), (50, 5), (300, 200), (1, 2)])
def test_pieces_of_prompts(dim, window, sinks):
    """More keys than queries, as many, and fewer: a query ahead of all keys sees none."""
    lengths, keys = [10, 300, 5, 40, 0, 7, 1], [1000, 431, 5, 3, 60, 0, 2000]
    q, k, v = inputs(lengths, keys, 4, 2, dim, 5)
    got = ops.prompt_attention(q, k, v, ends(lengths), window=window, sinks=sinks, k_offsets=ends(keys))
    check(got, q, k, v, lengths, keys, window, sinks)
    assert (got[315:352] == 0).all() and (got[355:362] == 0).all()
    ops.check_device_errors()


def test_no_keys_at_all():
    q = inputs([5], [5], 4, 2, 64, 1)[0]
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 3)
    got = ops.prompt_attention(q, none, none, ends([4]), k_offsets=ends([0]), out=out)
    assert (got[:4] == 0).all() and (got[4:] == 3).all()
    assert ops.prompt_attention(none, none, none, ends([0])).shape == (0, 2, 64)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 11, 27, 64, 65, 128, 129, 200])
def test_heads_of_a_group(group):
    lengths = [70, 3, 150]
    q, k, v = inputs(lengths, lengths, 2 * group, 2, 64, group)
    check(ops.prompt_attention(q, k, v, ends(lengths), window=40, sinks=2), q, k, v, lengths, lengths, 40, 2)
    ops.check_device_errors()


SPLIT = [([1], [5000], 8, 2, 128), ([70, 3], [3000, 9000], 8, 2, 64), ([3500], [3500], 4, 1, 128), ([1, 1, 130, 40, 0, 7], [14097, 1, 2222, 9001, 50, 5], 7, 1, 128),
         ([600, 300], [6600, 1300], 8, 8, 64), ([33], [20000], 2, 2, 128), ([5, 900], [3, 4000], 16, 1, 64)]


@pytest.mark.parametrize("lengths,keys,heads,kv_heads,dim", SPLIT)
@pytest.mark.parametrize("window,sinks", [(None, 0), (3000, 5), (2700, 300)])
def test_few_queries_with_many_keys(lengths, keys, heads, kv_heads, dim, window, sinks):
    """Most of them cut into parts that CTAs share."""
    q, k, v = inputs(lengths, keys, heads, kv_heads, dim, 7, behind=3)
    got = ops.prompt_attention(q, k, v, ends(lengths), window=window, sinks=sinks, k_offsets=ends(keys))
    check(got, q, k, v, lengths, keys, window, sinks)
    assert (got[sum(lengths):] == 0).all()
    assert torch.equal(got, ops.prompt_attention(q, k, v, ends(lengths), window=window, sinks=sinks, k_offsets=ends(keys)))
    ops.check_device_errors()


def test_which_are_cut():
    from sharq_b200 import _lib

    size = _lib.lib().sharq_prompt_attention_workspace_bytes
    cut = [size(sum(n), sum(m), heads, kv_heads, dim, len(n), 0, 0) > 0 for n, m, heads, kv_heads, dim in SPLIT]
    assert cut == [True, True, False, True, True, True, False]
    assert size(120, 9500, 4, 2, 128, 3, 0, 0) > 0 and size(300, 9000, 8, 2, 128, 2, 0, 0) > 0  # of the two tests below


def test_parts_with_values_that_are_not_finite_and_bad_offsets():
    lengths, keys = [40, 30, 50], [3000, 4000, 2500]
    q, k, v = inputs(lengths, keys, 4, 2, 128, 3)
    v[2990, 1, 5], v[3001, 0, 9], v[7100, 1, 3] = math.inf, math.nan, -math.inf
    got = ops.prompt_attention(q, k, v, ends(lengths), k_offsets=ends(keys))
    check(got, q, k, v, lengths, keys)
    q[45, 2, 3] = math.nan
    got = ops.prompt_attention(q, k, v, ends(lengths), k_offsets=ends(keys))
    assert got[45, 2].isnan().all()
    at = ends(keys)
    at[1] = 9501
    got = ops.prompt_attention(q, k, v, ends(lengths), k_offsets=at)
    with pytest.raises(RuntimeError, match="offsets"):
        ops.check_device_errors()
    assert got[:70].isnan().all() and not got[70:, :2].isnan().any()


def test_parts_in_a_graph_whose_lengths_change():
    q, k, v = inputs([300], [9000], 8, 2, 128, 4)
    at, keys = ends([200, 100]), ends([5000, 4000])
    ops.prompt_attention(q, k, v, at, k_offsets=keys)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.prompt_attention(q, k, v, at, k_offsets=keys)
    for lengths, m in (([299, 1], [300, 8700]), ([0, 300], [10, 8990]), ([100, 50], [9000, 0]), ([150, 150], [4500, 4500])):
        at.copy_(ends(lengths))
        keys.copy_(ends(m))
        graph.replay()
        check(got, q, k, v, lengths, m)
    ops.check_device_errors()


def test_an_output_at_any_multiple_of_16_bytes():
    lengths = [130, 70]
    q, k, v = inputs(lengths, lengths, 4, 2, 64, 5)
    want = ops.prompt_attention(q, k, v, ends(lengths))
    for shift in (8, 16, 24):
        out = torch.full((200 * 256 + 64,), 3.0, dtype=torch.bfloat16, device="cuda")
        ops.prompt_attention(q, k, v, ends(lengths), out=out[shift:shift + 200 * 256].view(200, 4, 64))
        assert torch.equal(out[shift:shift + 200 * 256].view(200, 4, 64), want) and (out[:shift] == 3).all() and (out[shift + 200 * 256:] == 3).all()
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.prompt_attention(q, k, v, ends(lengths), out=out[4:4 + 200 * 256].view(200, 4, 64))


def test_many_sequences():
    g = torch.Generator().manual_seed(3)
    lengths = (torch.rand(700, generator=g) ** 4 * 90).int().tolist()
    q, k, v = inputs(lengths, lengths, 4, 1, 64, 8)
    check(ops.prompt_attention(q, k, v, ends(lengths)), q, k, v, lengths, lengths)
    check(ops.prompt_attention(q, k, v, ends(lengths), window=7, sinks=1), q, k, v, lengths, lengths, 7, 1)


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0, 1e-6, 8.0])
def test_scales(scale):
    lengths = [300, 40]
    q, k, v = inputs(lengths, lengths, 4, 2, 128, 4)
    check(ops.prompt_attention(q, k, v, ends(lengths), scale=scale, window=77, sinks=3), q, k, v, lengths, lengths, 77, 3, scale=scale)


def test_scores_that_rise_and_values_of_all_sizes():
    """The maximum rises in every tile; values up to the largest, whose sums would overflow."""
    n = 1000
    q, k, v = inputs([n], [n], 2, 1, 128, 6)
    q[:] = 1
    k[:] = (torch.arange(n, device="cuda")[:, None, None] / 40).to(torch.bfloat16)
    v[::2] *= 2.0 ** 124
    v[1::4] *= 2.0 ** -120
    check(ops.prompt_attention(q, k, v, ends([n])), q, k, v, [n], [n])
    check(ops.prompt_attention(q, k, v, ends([n]), scale=-1.0), q, k, v, [n], [n], scale=-1.0)
    v[:] = torch.finfo(torch.bfloat16).max
    assert (ops.prompt_attention(q, k, v, ends([n]), scale=1e-3) == torch.finfo(torch.bfloat16).max).all()


@pytest.mark.parametrize("dim,group", [(128, 4), (64, 1)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_masked_places_that_are_not_finite(dim, group, value):
    """What a query does not see says nothing: keys and values of other sequences, behind the last one, after it, ahead of its window."""
    lengths = [150, 90, 200]
    for window, sinks in ((None, 0), (20, 3)):
        q, k, v = inputs(lengths, lengths, 2 * group, 2, dim, 9, behind=300)
        v[155, 0, 5] = value          # sequence 1, seen by nearly all of its queries, unless the window leaves it
        v[240 + 60, 1, dim - 1] = value  # sequence 2, in the middle
        v[149, 0, 17] = value         # the last of sequence 0
        k[240 + 199, 1, 3] = value
        got = ops.prompt_attention(q, k, v, ends(lengths), window=window, sinks=sinks)
        assert (got[440:] == 0).all()
        rows = torch.ones(440, dtype=torch.bool, device="cuda")
        rows[439] = False  # its own key is not finite: NaN in the heads that read it
        want, size, reach = definition64(q[:440], k, v, lengths, lengths, window or 0, sinks, dim ** -0.5)
        assert got[439, group:].isnan().all() or not got[439, group:].isnan().any()
        reach[439] = 0
        got, want, limit = got[:440].double()[rows], want[rows], bound(want, size, reach, dim, 200)[rows]
        fine = want.isfinite()
        assert torch.equal(fine, got.isfinite()) and torch.equal(want.isnan(), got.isnan()) and torch.equal(want[want.isinf()], got[got.isinf()])
        assert ((got - want).abs() <= limit)[fine].all()
    ops.check_device_errors()


def test_a_score_that_is_nan_spoils_its_row():
    q, k, v = inputs([300], [300], 2, 1, 128, 2)
    q[200, 1, 7] = math.nan
    got = ops.prompt_attention(q, k, v, ends([300]))
    assert got[200, 1].isnan().all()
    got[200, 1] = 0
    assert got.isfinite().all()


def test_rows_of_no_sequence():
    lengths = [40, 100]
    q, k, v = inputs(lengths, lengths, 4, 2, 128, 3, behind=77)
    at = ends(lengths)
    got = ops.prompt_attention(q, k, v, at, window=30, sinks=2)
    check(got, q, k, v, lengths, lengths, 30, 2)
    assert (got[140:] == 0).all()
    out = torch.full_like(got, 5)
    assert ops.prompt_attention(q, k, v, at, window=30, sinks=2, out=out) is out
    assert torch.equal(out[:140], got[:140]) and (out[140:] == 5).all()
    # rows ahead of the first sequence
    moved = [torch.cat((torch.full_like(x[:9], math.nan), x)) for x in (q, k, v)]
    got2 = ops.prompt_attention(*moved, at + 9, window=30, sinks=2)
    assert (got2[:9] == 0).all() and torch.equal(got2[9:], got)
    # a batch without tokens
    assert (ops.prompt_attention(q, k, v, torch.zeros(4, dtype=torch.int32, device="cuda")) == 0).all()
    ops.check_device_errors()


def test_strides():
    lengths = [90, 200]
    q, k, v = inputs(lengths, lengths, 6, 2, 128, 12)
    want = ops.prompt_attention(q, k, v, ends(lengths), window=60, sinks=4)
    by_head = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(want, ops.prompt_attention(*by_head, ends(lengths), window=60, sinks=4))
    merged = torch.cat([x.reshape(290, -1) for x in (q, k, v)], 1)
    parts = [p.view(290, -1, 128) for p in merged.split((768, 256, 256), 1)]
    assert torch.equal(want, ops.prompt_attention(*parts, ends(lengths), window=60, sinks=4))


def test_offsets_that_cannot_be():
    lengths = [60, 50, 70]
    q, k, v = inputs(lengths, lengths, 4, 2, 64, 13)
    good = ops.prompt_attention(q, k, v, ends(lengths))
    for bad in ([0, 60, 110, 181], [0, 60, 50, 180], [-1, 60, 110, 180], [0, 2 ** 31 - 1, 110, 180], [0, 60, -2 ** 31, 180]):
        at = torch.tensor(bad, dtype=torch.int32, device="cuda")
        got = ops.prompt_attention(q, k, v, at)
        with pytest.raises(RuntimeError, match="offsets"):
            ops.check_device_errors()
        for i in range(3):
            if 0 <= bad[i] <= bad[i + 1] <= 180 and (bad[i], bad[i + 1]) == (sum(lengths[:i]), sum(lengths[:i + 1])):
                assert torch.equal(got[bad[i]:bad[i + 1]], good[bad[i]:bad[i + 1]])
        got = ops.prompt_attention(q, k, v, ends(lengths), k_offsets=at)
        with pytest.raises(RuntimeError, match="offsets"):
            ops.check_device_errors()
        for i in range(3):
            rows = got[sum(lengths[:i]):sum(lengths[:i + 1])]
            assert rows.isnan().all() if not 0 <= bad[i] <= bad[i + 1] <= 180 else True
    assert torch.equal(good, ops.prompt_attention(q, k, v, ends(lengths)))
    ops.check_device_errors()


@pytest.mark.parametrize("bad,whole", [([0, 100, 60], (0, 100)), ([2 ** 31 - 1, 0, 50], (0, 50)), ([-7, 40, 130], (40, 130)), ([30, 130, -1], (30, 130))])
def test_rows_of_a_good_sequence_beside_bad_offsets(bad, whole):
    """They are neither zeros, as rows of no sequence, nor another sequence's."""
    n = whole[1] - whole[0]
    q, k, v = inputs([150], [150], 4, 2, 128, 15)
    rows = slice(*whole)
    want = ops.prompt_attention(*(x[rows].contiguous() for x in (q, k, v)), ends([n]), window=40, sinks=2)
    for _ in range(5):
        got = ops.prompt_attention(q, k, v, torch.tensor(bad, dtype=torch.int32, device="cuda"), window=40, sinks=2)
        assert torch.equal(got[rows], want) and (got[max(whole[1], *(x for x in bad if x <= 150)):] == 0).all()
        with pytest.raises(RuntimeError, match="offsets"):
            ops.check_device_errors()


def test_offsets_beyond_32_bits():
    """Elements of the activations beyond 2^31, and rows far into a sequence."""
    heads, dim, n = 160, 128, 110000
    q = torch.empty(n, heads, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    k, v = q[:, :20], q[:, 100:120]
    got = ops.prompt_attention(q, k, v, ends([n]), window=100, sinks=3)
    for p in (105, 1000, 104900, 109999):
        j = torch.tensor([0, 1, 2, *range(p - 99, p + 1)], device="cuda")
        a = torch.einsum("gd,jgd->gj", q[p].double(), k[j].double().repeat_interleave(8, 1)) * dim ** -0.5
        w = torch.softmax(a, -1)
        vv = v[j].double().repeat_interleave(8, 1)
        want, size = torch.einsum("gj,jgd->gd", w, vv), torch.einsum("gj,jgd->gd", w, vv.abs())
        reach = torch.einsum("gd,jgd->gj", q[p].double().abs(), k[j].double().abs().repeat_interleave(8, 1)).amax(-1)[:, None] * dim ** -0.5
        assert ((got[p].double() - want).abs() <= bound(want, size, reach, dim, 103)).all()
    ops.check_device_errors()


def test_two_calls_at_once():
    """On streams of their own, beside one another and beside a product that uses tensor memory too."""
    lengths = [[700, 90, 1200], [40] * 60]
    sets = [inputs(n, n, 8, 2, 128, 20 + i) for i, n in enumerate(lengths)]
    at = [ends(n) for n in lengths]
    want = [ops.prompt_attention(*x, at[i], window=300, sinks=4) for i, x in enumerate(sets)]
    w = torch.randn(1024, 512, device="cuda").to(torch.bfloat16)
    qw, sfs, sfd, scale = ops.scaled_quantize_w32_shared(w)
    x = torch.randn(300, 512, device="cuda").to(torch.bfloat16)
    product = ops.sharq_linear_forward(x, qw, sfs, sfd, float(scale))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = [[], [], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.prompt_attention(*sets[i], at[i], window=300, sinks=4))
        with torch.cuda.stream(streams[2]):
            got[2].append(ops.sharq_linear_forward(x, qw, sfs, sfd, float(scale)))
    torch.cuda.synchronize()
    for a, b in zip(got, (*want, product)):
        assert all(torch.equal(y, b) for y in a)
    ops.check_device_errors()


def test_captured_and_on_another_stream():
    lengths = [100, 300]
    q, k, v = inputs(lengths, lengths, 4, 2, 128, 14)
    at = ends(lengths)
    want = ops.prompt_attention(q, k, v, at, window=50, sinks=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.prompt_attention(q, k, v, at, window=50, sinks=4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.prompt_attention(q, k, v, at, window=50, sinks=4)
    at.copy_(ends([250, 150]))
    v.mul_(2)
    graph.replay()
    assert torch.equal(got, ops.prompt_attention(q, k, v, ends([250, 150]), window=50, sinks=4))
    ops.check_device_errors()


def test_refusals():
    lengths = [30, 20]
    q, k, v = inputs(lengths, lengths, 4, 2, 64, 1)
    at = ends(lengths)
    wide = torch.zeros(50, 4, 96, dtype=torch.bfloat16, device="cuda")
    good = dict(q=q, k=k, v=v, offsets=at)
    ops.prompt_attention(**good)
    for changes in (dict(q=q.float()), dict(q=q[0]), dict(k=k.half()), dict(k=k[:49]), dict(v=v[:, :1]), dict(v=v.cpu()), dict(q=q[:, :3]), dict(k=k.transpose(1, 2)),
                    dict(q=wide, k=wide[:, :2], v=wide[:, :2]), dict(offsets=at.long()), dict(offsets=at[:1]), dict(offsets=at.cpu()), dict(offsets=at[None]),
                    dict(k_offsets=at[:2]), dict(k_offsets=at.long()), dict(window=0), dict(window=-3), dict(sinks=-1), dict(out=q[:, :2]), dict(out=q.float()),
                    dict(out=torch.empty(4, 50, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)), dict(k=k[:, :1].expand(50, 2, 64)),
                    dict(q=torch.zeros(50, 4, 68, dtype=torch.bfloat16, device="cuda")[:, :, :64])):
        with pytest.raises(RuntimeError):
            ops.prompt_attention(**{**good, **changes})
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.prompt_attention(q.cpu(), k, v, at)
    ops.check_device_errors()
