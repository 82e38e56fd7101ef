"""Decode steps of the quantised decoder against values of their own: the layers from their definition in 64 bits, on the weights that the
4-bit payloads stand for (the oracle's dequantisation), and the decoder's other paths where these give the same."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def small(**kw):
    from sharq_b200.decoder import DecoderConfig

    return DecoderConfig(**{**dict(hidden=512, layers=1, heads=8, kv_heads=2, head_dim=128, ffn=1024, vocab=2000), **kw})


def draw(cfg, *shape):
    return torch.randint(0, cfg.vocab, shape, generator=torch.Generator().manual_seed(1)).cuda()


def weight(oracle, layer):
    """What a SHARQ layer multiplies with, float64 [out, in]."""
    q, sf = layer.weight_q.cpu().numpy(), layer.scale_w_dense.cpu().numpy()
    return torch.from_numpy(oracle.dequant_dense(q, sf, 16)).cuda().double() * layer.weight_scale_host


def logits64(oracle, model, ids, cos, sin, mistake=None):
    """Logits [B, S, vocab] behind every token, from the definition, in 64 bits.  mistake: a fault that the comparison has to see."""
    cfg = model.cfg
    b, s = ids.shape
    d, heads, kv = cfg.head_dim, cfg.heads, cfg.kv_heads
    cos, sin = (t[:s].double()[None, :, None] for t in (cos, sin))
    reach = torch.ones(s, s, dtype=torch.bool, device=ids.device).tril(-1 if mistake == "length" else 0)

    def norm(x, w):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.eps) * w.double()

    def turn(x):
        return x * cos + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1) * sin

    x = model.embed[ids].double()
    for layer in model.layers:
        first, second = layer.input_norm, layer.post_norm
        if mistake == "norms":
            first, second = second, first
        qkv = norm(x, first) @ weight(oracle, layer.qkv).T
        if layer.qkv.bias is not None and mistake != "bias":
            qkv = qkv + layer.qkv.bias.double()
        q, k, v = qkv.view(b, s, -1, d).split((heads, kv, kv), 2)
        at = torch.arange(heads, device=ids.device) // (heads // kv)
        if mistake == "heads":
            at = torch.arange(heads, device=ids.device) % kv
        score = torch.einsum("bqhd,bkhd->bhqk", turn(q), turn(k)[:, :, at]) * d ** -0.5
        p = torch.softmax(score.masked_fill(~reach, -torch.inf), -1).nan_to_num(0)
        o = torch.einsum("bhqk,bkhd->bqhd", p, v[:, :, at]).reshape(b, s, heads * d) @ weight(oracle, layer.o_proj.local).T
        mid = o if mistake == "residual" else x + o
        gate, up = (norm(mid, second) @ weight(oracle, layer.gate_up).T).chunk(2, -1)
        if mistake == "swapped":
            gate, up = up, gate
        x = (mid if mistake != "addend" else x) + (torch.nn.functional.silu(gate) * up) @ weight(oracle, layer.down.local).T
    return norm(x, model.final_norm) @ model.lm_head.double().T


def roundings(cfg):
    """Roundings to bf16 (2^-8 of the value at most) that follow one another on the way to a logit: norm, projection, rotation, attention, output
    projection, sum, norm, gate and up (a factor each), SwiGLU, down projection and sum of a layer, the last norm and the logit."""
    return (12 * cfg.layers + 2) * 2.0 ** -8


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("kw", [dict(), dict(qkv_bias=True), dict(head_dim=64, heads=4, kv_heads=4), dict(layers=2), dict(layers=2, qkv_bias=True)])
def test_weight_only_decode_gives_the_values_of_its_weights(oracle, kw):
    """From the first token on, every logit within the roundings of the steps in between; and the comparison sees mistakes: each of them
    moves the values by more than twice that."""
    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg = small(**kw)
    model = SharqDecoder(cfg, torch.device("cuda"), seed=7)
    if cfg.qkv_bias:
        for layer in model.layers:
            layer.qkv.bias *= 20  # of the size of what it is added to
    ids = draw(cfg, 3, 6)
    cache = model.new_cache(3, 20, page_size=4)
    got = torch.stack([model.decode(ids[:, i], cache, weight_only=True) for i in range(6)], 1)
    ops.check_device_errors()
    want = logits64(oracle, model, ids, cache.cos, cache.sin)
    for i in range(6):
        assert off(got[:, i], want[:, i]) <= roundings(cfg), i
    # (a bias of that size leaves the FFN little to say)
    mistakes = ["bias", "length"] if cfg.qkv_bias else ["swapped", "residual", "addend", "length"] + ["norms"] * (cfg.layers == 1)
    mistakes += ["heads"] * (cfg.heads != cfg.kv_heads)
    for mistake in mistakes:
        wrong = logits64(oracle, model, ids, cache.cos, cache.sin, mistake)
        assert off(wrong, want) > 2 * roundings(cfg), mistake


@pytest.mark.parametrize("kw", [dict(layers=2), dict(qkv_bias=True), dict(head_dim=64, heads=4, kv_heads=4), dict(layers=2, experts=4)])
@pytest.mark.parametrize("rows", [1, 3])
def test_quantised_decode_of_a_first_token_is_its_prefill(rows, kw):
    """Attention over one token gives its value, so both paths have the same inputs to every product: the same bits."""
    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg = small(**kw)
    model = SharqDecoder(cfg, torch.device("cuda"), seed=7)
    ids = draw(cfg, rows, 1)
    want = model.prefill(ids)
    assert torch.equal(model.decode(ids[:, 0], model.new_cache(rows, 20)), want)
    assert torch.equal(model.prefill(ids, cache=model.new_cache(rows, 20)), want)
    ops.check_device_errors()


@pytest.mark.parametrize("weight_only", [False, True])
def test_quantised_decode_tracks_the_unquantised_prompt(weight_only):
    """A token behind a quantised prompt, as close to the unquantised layers as a quantised prompt has to be."""
    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg = small(layers=2, heads=4)
    model = SharqDecoder(cfg, torch.device("cuda"), keep_reference=True, seed=3)
    ids = draw(cfg, 2, 160)
    cache = model.new_cache(2, 200)
    model.prefill(ids[:, :159], cache=cache)
    got = model.decode(ids[:, 159], cache, weight_only=weight_only)
    ops.check_device_errors()
    want = model.prefill(ids, reference=True)
    assert off(got, want.double()) < 0.35
    assert torch.nn.functional.cosine_similarity(got.flatten(), want.flatten(), dim=0) > 0.93


@pytest.mark.parametrize("qkv_bias", [False, True])
def test_two_ranks_give_the_values_of_one(oracle, qkv_bias):
    """Ranks as threads of one process; a partial sum is rounded once more (two of them in place of one: 2 more per sum at most)."""
    from sharq_b200 import ops
    from sharq_b200.decoder import SharqDecoder

    cfg, world, dev = small(layers=2, qkv_bias=qkv_bias), 2, torch.device("cuda")
    ids = draw(cfg, 3, 5)
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
            cache = model.new_cache(3, 20)
            results[rank] = torch.stack([model.decode(ids[:, i], cache, weight_only=True) for i in range(5)], 1)
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
    one = SharqDecoder(cfg, dev, seed=11)
    cache = one.new_cache(3, 20)
    want = logits64(oracle, one, ids, cache.cos, cache.sin)
    assert torch.equal(results[0], results[1])
    assert off(results[0], want) <= roundings(cfg) + 4 * 2 * 2.0 ** -8


def test_products_stand_for_the_oracles_weights(oracle):
    """weight_only_linear against the oracle's dequantisation of the same buffers, for both kinds of weight."""
    from sharq_b200 import ops
    from tests.test_weight_only_gpu import check

    g = torch.Generator().manual_seed(2)
    w = (0.02 * torch.randn(392, 896, generator=g)).to(torch.bfloat16).cuda()
    x = torch.randn(5, 896, generator=g).to(torch.bfloat16).cuda()
    q, _, sfd, scale = ops.scaled_quantize_w32_shared(w)
    for q, sf, scale in ((q, sfd, scale), ops.scaled_quantize_nvfp4(w)):
        held = torch.from_numpy(oracle.dequant_dense(q.cpu().numpy(), sf.cpu().numpy(), 16)).cuda().double()
        check(ops.weight_only_linear(x, q, sf, scale), x, held, float(scale))
        # and the weight itself, to a sixth of a block's largest element (half the widest step of e2m1, 4 to 6) and its scale's rounding (2^-4)
        block = w.double().view(392, 28, 32).abs().amax(-1, keepdim=True).expand(-1, -1, 32).reshape(392, 896)
        assert bool(((held * float(scale) - w.double()).abs() <= (1 / 6 + 2.0 ** -4 + 2.0 ** -7) * block + 2.0 ** -10 * 6 * float(scale)).all())
