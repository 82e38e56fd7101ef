"""Decode steps of the decoder stack: the new operators one behind the other, as a model calls them."""
import pytest
import torch

from tests import paged_util as P
from tests.test_weight_only_gpu import check as check_product, weight64

pytestmark = pytest.mark.gpu


def small(**kw):
    from sharq_b200.decoder import DecoderConfig

    return DecoderConfig(**{**dict(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=128, ffn=1024, vocab=2000), **kw})


def tokens(cfg, *shape, seed=0):
    return torch.randint(0, cfg.vocab, shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page_size", [16, 24])
def test_projection_append_attention_projection(fp8, page_size):
    """The operators of a layer's attention block over several steps, each against its definition in 64 bits on the inputs that it had:
    ragged prompts, then single tokens, one sequence behind the others."""
    from sharq_b200 import ops

    seqs, heads, kv, dim, hidden, steps = 3, 8, 2, 128, 512, 5
    g = torch.Generator().manual_seed(1)
    w = [ops.scaled_quantize_w32_shared((0.03 * torch.randn(n, k, generator=g)).to(torch.bfloat16).cuda())
         for n, k in (((heads + 2 * kv) * dim, hidden), (hidden, heads * dim))]
    (qw, _, qsf, qscale), (ow, _, osf, oscale) = w
    prompts = [7, 40, 1]
    table, pages = P.make_table([n + steps for n in prompts], page_size, 1, 3)
    cache = P.make_cache(pages, kv, page_size, dim, fp8, 5)
    scales = dict(k_scale=cache[2], v_scale=cache[3])
    cos, sin = P.rope_tables(64, dim)
    held_k, held_v = ([[] for _ in prompts] for _ in range(2))  # what every sequence has been given, in 64 bits

    def keep(q, rows, sequences, positions, qkv):
        want_q, want_k, want_v = P.rotated64(qkv, heads, kv, dim, cos, sin, positions)
        assert bool(((q.double() - want_q).abs() <= 2.0 ** -8 * (1 + 2.0 ** -15) * want_q.abs()).all())
        for c, want, scale, held in zip(cache[:2], (want_k, want_v), cache[2:], (held_k, held_v)):
            got = c[table[sequences.long(), (positions // page_size).long()].long(), :, (positions % page_size).long()]
            if fp8:
                want = (want / scale.double()[:, None]).clamp(-448, 448)
                bound = 2.0 ** -4 * (1 + 2.0 ** -15) * want.abs() + 2.0 ** -10
            else:
                bound = 2.0 ** -8 * (1 + 2.0 ** -15) * want.abs()
            assert bool(((got.double() - want).abs() <= bound).all())
            for row, s in enumerate(sequences.tolist()):
                held[s].append(got[row].double() * (scale.double()[:, None] if fp8 else 1))

    sequences = torch.cat([torch.full((n,), i) for i, n in enumerate(prompts)]).to(torch.int32).cuda()
    positions = torch.cat([torch.arange(n) for n in prompts]).to(torch.int32).cuda()
    qkv = torch.randn(sum(prompts), (heads + 2 * kv) * dim, generator=g).to(torch.bfloat16).cuda()
    q = ops.rope_append_paged(qkv, heads, kv, dim, cos, sin, positions, table, *cache[:2], sequences=sequences, **scales)
    keep(q, len(sequences), sequences, positions, qkv)
    for step in range(steps):
        x = torch.randn(seqs, hidden, generator=g).to(torch.bfloat16).cuda()
        qkv = ops.weight_only_linear(x, qw, qsf, qscale)
        check_product(qkv, x, weight64(qw, qsf), float(qscale))
        positions = torch.tensor([n + step for n in prompts], dtype=torch.int32).cuda()
        q = ops.rope_append_paged(qkv, heads, kv, dim, cos, sin, positions, table, *cache[:2], **scales)
        keep(q, seqs, torch.arange(seqs, dtype=torch.int32).cuda(), positions, qkv)
        out = ops.paged_attention(q, *cache[:2], table, positions + 1, **scales)
        for s in range(seqs):
            k64, v64 = (torch.stack(h[s], 1) for h in (held_k, held_v))  # [kv, tokens, dim]
            n = k64.shape[1]
            ident = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
            want, size, reach = P.attention64(q[s:s + 1], k64[None], v64[None], ident, [n])
            bound = P.attention_bound(want, size, reach, dim, n, fp8)
            assert bool(((out[s:s + 1].double() - want).abs() <= bound).all())
        a = out.view(seqs, heads * dim)
        check_product(ops.weight_only_linear(a, ow, osf, oscale), a, weight64(ow, osf), float(oscale))
    ops.check_device_errors()


@pytest.mark.parametrize("kw", [dict(), dict(qkv_bias=True), dict(head_dim=64, heads=4, kv_heads=4), dict(experts=4, top_k=2)])
def test_decode_follows_prefill(kw):
    """Tokens after a prompt give what the prompt with those tokens gives.  With unquantised layers the two differ by roundings of the
    residual stream and of attention, some twenty of half a step (2^-8) in sequence over the two layers: at most 8 %."""
    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg = small(**kw)
    model = SharqDecoder(cfg, torch.device("cuda"), keep_reference=True, seed=3)
    ids = tokens(cfg, 3, 80)
    reference = cfg.experts == 0  # a nearly tied router may send a token elsewhere for a rounding
    cache = model.new_cache(3, 100, page_size=16)
    model.prefill(ids[:, :75], reference=reference, cache=cache)
    for i in range(75, 80):
        got = model.decode(ids[:, i], cache, reference=reference)
        assert got.shape == (3, cfg.vocab) and bool(torch.isfinite(got).all())
    ops.check_device_errors()
    assert cache.lengths == [80] * 3 and cache.device_lengths.tolist() == [80] * 3
    if reference:
        want = model.prefill(ids, reference=True)
        assert (got - want).norm() <= 0.08 * want.norm()
    # a cache does not change the prompt's own attention: the same layers, rotated with one rounding instead of three
    with pytest.raises(ValueError, match="empty cache"):
        model.prefill(ids, cache=cache)


@pytest.mark.parametrize("weight_only", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_quantised_decode_eager_and_captured(weight_only, dtype):
    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg = small()
    model = SharqDecoder(cfg, torch.device("cuda"), seed=3)
    ids = tokens(cfg, 2, 40)
    scale = None if dtype == torch.bfloat16 else torch.full((2, 2), 0.02)
    caches = [model.new_cache(2, 64, page_size=16, dtype=dtype, k_scale=scale, v_scale=scale) for _ in range(2)]
    for cache in caches:
        model.prefill(ids[:, :35], cache=cache)
    eager = [model.decode(ids[:, i], caches[0], weight_only=weight_only).clone() for i in range(35, 40)]
    cache = caches[1]
    cache.reserve([5, 5])
    token, positions, lengths = ids[:, 35].clone(), cache.device_lengths.clone(), cache.device_lengths + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the first token, and the warm-up
        model.decode_step(token, cache, positions, lengths, weight_only=weight_only)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.decode_step(token, cache, positions, lengths, weight_only=weight_only)
    for i, want in zip(range(35, 40), eager):
        token.copy_(ids[:, i])
        positions.fill_(i)
        lengths.fill_(i + 1)
        graph.replay()
        assert torch.equal(logits, want)
    ops.check_device_errors()


def test_decode_under_tensor_parallelism():
    """Two ranks as threads of one process, their partial sums exchanged on the host: each keeps its own heads' cache."""
    import threading

    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg, world, dev = small(), 2, torch.device("cuda")
    ids = tokens(cfg, 2, 30)
    barrier, parts, results, errors = threading.Barrier(world), [None] * world, [None] * world, []

    def hook_for(rank):
        def hook(t):
            torch.cuda.synchronize()
            parts[rank] = t
            barrier.wait()
            total = torch.stack([p.float() for p in parts]).sum(0).to(torch.bfloat16)
            torch.cuda.synchronize()
            barrier.wait()
            return total
        return hook

    def run(rank):
        try:
            torch.cuda.set_device(0)
            model = SharqDecoder(cfg, dev, world=world, rank=rank, seed=11, reduce_hook=hook_for(rank))
            cache = model.new_cache(2, 64)
            model.prefill(ids[:, :29], cache=cache)
            assert cache.k.shape[2] == 1
            results[rank] = [model.decode(ids[:, 29], cache, weight_only=True).clone()]
            torch.cuda.synchronize()
        except Exception as exc:  # release the other instead of leaving it at the barrier
            errors.append(exc)
            barrier.abort()

    threads = [threading.Thread(target=run, args=(r,)) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=300)
    assert not errors, errors
    ops.check_device_errors()
    assert torch.equal(results[0][0], results[1][0]) and bool(torch.isfinite(results[0][0]).all())


def test_refusals_of_the_model():
    from sharq_b200.decoder import SharqDecoder

    cfg = small()
    model = SharqDecoder(cfg, torch.device("cuda"), seed=3)
    ids = tokens(cfg, 17, 3)
    cache = model.new_cache(17, 4, page_size=4)
    with pytest.raises(ValueError, match="sequence for every prompt"):
        model.prefill(ids[:2], cache=cache)
    model.prefill(ids, cache=cache)
    with pytest.raises(ValueError, match="one token for every"):
        model.decode(ids[:3, 0], cache)
    with pytest.raises(ValueError, match="at most 16 sequences"):
        model.decode(ids[:, 0], cache, weight_only=True)
    model.decode(ids[:, 0], cache)
    with pytest.raises(RuntimeError, match="does not fit"):
        model.decode(ids[:, 0], cache)
    assert cache.lengths == [4] * 17
    plain = SharqDecoder(cfg, torch.device("cuda"), seed=3, mode="BF16")
    cache = plain.new_cache(1, 8)
    plain.prefill(ids[:1], cache=cache)
    with pytest.raises(ValueError, match="SHARQ mode"):
        plain.decode(ids[:1, 0], cache, weight_only=True)
    assert bool(torch.isfinite(plain.decode(ids[:1, 0], cache)).all())
