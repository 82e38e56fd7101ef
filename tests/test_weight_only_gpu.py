"""Products of unquantised rows with 4-bit weights against their definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def weight64(qw, sf):
    """What a payload and its dense scale factors stand for, float64 [N, K]."""
    n, k = qw.shape[0], qw.shape[1] * 2
    value = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=qw.device)
    w = value[torch.stack((qw & 15, qw >> 4), -1).view(n, k).long()]
    row, group = torch.arange(n, device=qw.device)[:, None], torch.arange(k // 16, device=qw.device)[None]
    at = (row // 128) * (k // 64) * 512 + (group // 4) * 512 + (row % 32) * 16 + (row // 32 % 4) * 4 + group % 4
    return w * sf.view(torch.float8_e4m3fn).double()[at].repeat_interleave(16, 1)


def random_weight(n, k, seed):
    """Every code and every scale factor but NaN."""
    g = torch.Generator().manual_seed(seed)
    qw = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=g)
    sf = torch.randint(0, 127, ((n // 128 + 1) * 128 * k // 16,), dtype=torch.uint8, generator=g)
    return qw.cuda(), sf.cuda()


def check(got, x, w, scale, bias=None):
    """got against bf16(scale * x . w^T + bias).  A float sum of exact products: the tensor core's over blocks of 128 (24 roundings of
    2^-23 at most) and one more per block, the factors' and the bias's roundings, in units of the sum of sizes; elements of x below 2^-39 of
    their block's largest may be lost; one rounding to bf16 (2^-8)."""
    xd = x.double()
    want = xd @ w.T * scale + (0 if bias is None else bias.double())
    size = xd.abs() @ w.abs().T * abs(scale) + (0 if bias is None else bias.double().abs())
    lost = 2.0 ** -39 * xd.abs().amax(1, keepdim=True) * w.abs().sum(1) * abs(scale)
    bound = (x.shape[1] / 128 + 32) * 2.0 ** -23 * size + lost + 2.0 ** -8 * (1 + 2.0 ** -7) * want.abs() + 1e-37
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


SHAPES = [(1, 4096, 4096), (16, 128, 64), (3, 1, 64), (8, 130, 192), (9, 257, 14336), (5, 1000, 18944), (16, 4608, 3584), (1, 128, 128),
          (7, 37888, 256), (2, 300, 320), (13, 129, 4032), (1, 64, 32768), (4, 40000, 448),
          (16, 136, 65536), (3, 200, 36864), (2, 5000, 512)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(m, n, k):
    from sharq_b200 import ops

    g = torch.Generator().manual_seed(m + n + k)
    qw, sf = random_weight(n, k, m)
    w = weight64(qw, sf)
    x = torch.randn(m, k, generator=g)
    x[:, ::97] *= 20
    x = x.to(torch.bfloat16).cuda()
    bias = torch.randn(n, generator=g).to(torch.bfloat16).cuda()
    got = ops.weight_only_linear(x, qw, sf, 0.37)
    check(got, x, w, float(torch.tensor(0.37)))
    scale = torch.tensor([0.011], device="cuda")
    check(ops.weight_only_linear(x, qw, sf, scale, bias=bias), x, w, float(scale), bias)
    # the same bits again, into a given tensor, from rows that are not contiguous
    wide = torch.zeros(m, k + 40, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:k + 8] = x
    out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    assert ops.weight_only_linear(wide[:, 8:k + 8], qw, sf, 0.37, out=out) is not None
    assert torch.equal(out, got)


def test_weights_as_the_package_quantises_them():
    from sharq_b200 import ops

    w = (0.02 * torch.randn(384, 512, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16).cuda()
    x = torch.randn(4, 512, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    q, _, sfd, scale = ops.scaled_quantize_w32_shared(w)
    check(ops.weight_only_linear(x, q, sfd, scale), x, weight64(q, sfd), float(scale))
    q, sf, scale = ops.scaled_quantize_nvfp4(w)
    check(ops.weight_only_linear(x, q, sf, scale), x, weight64(q, sf), float(scale))


def test_activations_of_every_size():
    """Powers of two over bf16's whole range in one row and one power per block, zeros, subnormal values, the largest."""
    from sharq_b200 import ops

    n, k = 200, 1024
    qw, sf = random_weight(n, k, 3)
    sf = sf.clamp(max=60)
    w = weight64(qw, sf)
    rows = [torch.zeros(k), torch.full((k,), 1e-40), torch.full((k,), 3e38), 2.0 ** (torch.arange(k) % 250 - 126).float(),
            2.0 ** (torch.arange(k) // 128 * 30 - 120).float(), torch.randn(k) * 1e-38]
    x = torch.stack(rows).to(torch.bfloat16).cuda()
    x[:, 1::2] *= -1
    check(ops.weight_only_linear(x, qw, sf, 2.0 ** -10), x, w, 2.0 ** -10)


def test_infinities_and_nan_stay_in_their_rows():
    from sharq_b200 import ops

    n, k = 200, 512
    qw, sf = random_weight(n, k, 3)
    w = weight64(qw, sf)
    x = torch.randn(6, k, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    x[1, 7] = float("inf")
    x[2, 300] = -float("inf")
    x[3, 511] = float("nan")
    x[4, 0], x[4, 400] = float("inf"), float("inf")
    x[5, 3], x[5, 5] = 3e38, -float("inf")
    got = ops.weight_only_linear(x, qw, sf, 1.0)
    want = x.double() @ w.T
    for i in range(6):
        assert torch.equal(got[i].isnan(), want[i].isnan()), i
    inf = want.isinf()
    assert torch.equal(got[inf].double(), want[inf])
    check(got[:1], x[:1], w, 1.0)


def test_layer_forward_weight_only_and_graphs():
    from sharq_b200 import ops
    from sharq_b200.qlinear import QLinearLayer

    g = torch.Generator().manual_seed(5)
    lin = torch.nn.Linear(256, 320, bias=True)
    x = torch.randn(2, 3, 256, generator=g).to(torch.bfloat16).cuda()
    for kind in ("SHARQ", "NVFP4"):
        layer = QLinearLayer(lin, quant_type=kind, device="cuda")
        got = layer.forward_weight_only(x)
        assert got.shape == (2, 3, 320)
        sf = layer.scale_w_dense if kind == "SHARQ" else layer.scale_w
        check(got.view(6, 320), x.view(6, 256), weight64(layer.weight_q, sf), layer.weight_scale_host, layer.bias)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.forward_weight_only(x)
        graph.replay()
        assert torch.equal(y, got)
        with pytest.raises(RuntimeError, match="at most 16 rows"):
            layer.forward_weight_only(x.expand(7, 2, 3, 256))
    ops.check_device_errors()


def test_refusals():
    from sharq_b200 import ops

    qw, sf = random_weight(128, 256, 1)
    x = torch.zeros(2, 256, dtype=torch.bfloat16).cuda()

    def refuse(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            ops.weight_only_linear(*args, **kw)

    refuse("CUDA bfloat16", x.float(), qw, sf, 1.0)
    refuse("CUDA bfloat16", x.cpu(), qw, sf, 1.0)
    refuse("unit column stride", x.t().contiguous().t(), qw, sf, 1.0)
    refuse("K/2 = 128", x, qw[:, :64].contiguous(), sf, 1.0)
    refuse("multiple of 64", x[:, :32].contiguous(), qw[:, :16].contiguous(), sf, 1.0)
    refuse("at most 16 rows", x[:1].expand(17, 256).contiguous(), qw, sf, 1.0)
    refuse("qw must be", x, qw.to(torch.int8), sf, 1.0)
    refuse("qw must be", x, qw.t().contiguous().t(), sf, 1.0)
    refuse("sfw_dense must be", x, qw, sf[:-1], 1.0)
    refuse("weight_scale", x, qw, sf, torch.ones(2).cuda())
    refuse("weight_scale", x, qw, sf, torch.ones(1))
    refuse("bias", x, qw, sf, 1.0, bias=torch.zeros(127, dtype=torch.bfloat16).cuda())
    refuse("out must be", x, qw, sf, 1.0, out=torch.zeros(2, 128).cuda())
    refuse("must not overlap", x[:1].expand(2, 256), qw, sf, 1.0)
    refuse("16-byte aligned", torch.zeros(2, 260, dtype=torch.bfloat16).cuda().view(-1)[4:516].view(2, 256), qw, sf, 1.0)
    assert ops.weight_only_linear(x[:0], qw, sf, 1.0).shape == (0, 128)


def test_layer_takes_activations_of_any_stride():
    from sharq_b200.qlinear import QLinearLayer

    g = torch.Generator().manual_seed(2)
    w = torch.nn.Linear(192, 40, bias=True)
    w.weight.data = (0.05 * torch.randn(40, 192, generator=g))
    layer = QLinearLayer(w.to(torch.bfloat16).cuda(), quant_type="SHARQ")
    x = torch.randn(192, 6, generator=g).to(torch.bfloat16).cuda().t()
    whole = torch.randn(5, 200, generator=g).to(torch.bfloat16).cuda()
    for strided in (x, whole[:, 3:195], whole[:1, 3:195].expand(4, 192)):
        assert torch.equal(layer.forward_weight_only(strided), layer.forward_weight_only(strided.clone(memory_format=torch.contiguous_format)))


# shares of the rows whose sums are joined in several turns, in one CTA and in clusters, beginning and ending within a pair of tiles
@pytest.mark.parametrize("m,n,k", [(8, 20000, 4096), (7, 28701, 4096), (16, 20000, 4096), (15, 9002, 14336), (9, 12345, 2048), (4, 16000, 8192),
                                   (2, 30000, 14336), (16, 20000, 512), (11, 3001, 20480)])
def test_products_joined_in_turns(m, n, k):
    from sharq_b200 import ops

    g = torch.Generator().manual_seed(m + n + k)
    qw, sf = random_weight(n, k, m + n + k)
    x = torch.randn(m, k, generator=g).to(torch.bfloat16).cuda()
    bias = torch.randn(n, generator=g).to(torch.bfloat16).cuda() if m % 2 else None
    got = ops.weight_only_linear(x, qw, sf, 0.25, bias=bias)
    ops.check_device_errors()
    for i in range(0, n, 4096):  # in pieces of whole blocks of 128 rows
        rows = min(4096, n - i)
        w = weight64(qw[i:i + rows], sf[i * k // 16:])
        check(got[:, i:i + rows], x, w, 0.25, None if bias is None else bias[i:i + rows])
    assert torch.equal(ops.weight_only_linear(x, qw, sf, 0.25, bias=bias), got)


@pytest.mark.parametrize("m,n", [(1, 4096), (1, 4098), (12, 512)])
def test_results_and_biases_at_any_element(m, n):
    from sharq_b200 import ops

    qw, sf = random_weight(n, 512, 3)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(m, 512, generator=g).to(torch.bfloat16).cuda()
    bias = torch.randn(n + 1, generator=g).to(torch.bfloat16).cuda()
    want = ops.weight_only_linear(x, qw, sf, 0.5, bias=bias[1:].clone())
    for shift in (0, 1, 2):
        room = torch.full((m * n + 8,), 7.0, dtype=torch.bfloat16, device="cuda")
        out = room[shift:shift + m * n].view(m, n)
        assert ops.weight_only_linear(x, qw, sf, 0.5, bias=bias[1:], out=out) is not None
        assert torch.equal(out, want)
        assert bool((room[:shift] == 7).all()) and bool((room[shift + m * n:] == 7).all())


@pytest.mark.parametrize("shape", [(0, 256), (2, 0, 256), (256,), (1, 1, 3, 256)])
def test_layer_forward_of_every_shape(shape):
    """No rows, a single one without a dimension of its own, and several dimensions."""
    from sharq_b200.qlinear import QLinearLayer

    layer = QLinearLayer(torch.nn.Linear(256, 320, bias=True), quant_type="SHARQ", device="cuda")
    x = torch.randn(shape, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    got = layer.forward_weight_only(x)
    assert got.shape == (*shape[:-1], 320)
    assert torch.equal(got.reshape(-1, 320), layer.forward_weight_only(x.reshape(-1, 256)))
