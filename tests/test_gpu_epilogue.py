"""Bias, activation and residual in the epilogue of a hybrid linear (`DualLinear.linear`, `run_packed`) against 64-bit arithmetic.

Tolerances: the sum over K is fp32 (K roundings of 2^-23 of the sum of its terms' sizes at most), bias, activation and residual add four
roundings of 2^-23 and the functions' own few units (2^-20 of their argument and value; no activation's slope exceeds 1.13), and one
rounding to 16 bits comes last.
"""
import math

import pytest
import torch

import oracle
from hygemm_vllm import native, producer
from hygemm_vllm.cache import PagedCache
from test_gpu_cache import bounds, check_packed
from test_gpu_cache import reference as attention_reference

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
REFERENCE = {
    None: lambda v: v,
    "relu": lambda v: v.clamp(min=0),
    "silu": lambda v: v * torch.sigmoid(v),
    "gelu": lambda v: 0.5 * v * (1 + torch.erf(v / math.sqrt(2))),
    "gelu_tanh": lambda v: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))),
}


def weights_of(layer):
    """The values a layer's codes stand for, in 64 bits."""
    w = torch.empty(layer.outputs, layer.k, dtype=torch.float64, device="cuda")
    for ids, codes, scales, fp4 in ((layer.lo, layer.w4, layer.sf4, True), (layer.hi, layer.w8, layer.sf8, False)):
        if ids.numel():
            w[ids.long()] = torch.from_numpy(oracle.decode(codes.cpu().numpy(), scales.cpu().numpy(), layer.k, fp4=fp4)).double().cuda()
    return w


def activations_of(x):
    q, sf = native.pack(x)
    return torch.from_numpy(oracle.decode(q.cpu().numpy(), sf.cpu().numpy(), x.shape[1], fp4=False)).double().cuda()


def check(y, layer, weights, x, bias, activation, residual):
    values = activations_of(x)
    total, size = values @ weights.T, values.abs() @ weights.abs().T
    if bias is not None:
        total, size = total + bias.double(), size + bias.double().abs()
    want = REFERENCE[activation](total)
    if residual is not None:
        want, size = want + residual.double(), size + residual.double().abs()
    fp32 = 1.2 * (layer.k * 2.0 ** -23 + 2.0 ** -20) * size
    assert y.dtype == layer.dtype
    assert bool(((y.double() - want).abs() <= torch.finfo(y.dtype).eps / 2 * (want.abs() + fp32) + fp32).all())


def make(outputs, k, high, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    weight = (0.05 * torch.randn(outputs, k, device="cuda", generator=g)).to(dtype)
    ids = torch.sort(torch.randperm(outputs, device="cuda", generator=g)[:high]).values
    return native.DualLinear(weight, ids), g


# outputs, k, high: one tile and less, odd sizes, K split over a cluster, several tiles a CTA, one partition alone
SHAPES = [(96, 128, 10), (385, 640, 41), (700, 3584, 128), (4864, 896, 486), (1024, 18944, 128), (256, 384, 0), (130, 256, 130), (9001, 512, 900)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_linear(shape, dtype):
    outputs, k, high = shape
    layer, g = make(outputs, k, high, dtype)
    weights = weights_of(layer)
    for n, tokens in enumerate((1, 7, 16, 17, 37, 64, 128, 129, 300, 777)):
        x = torch.randn(tokens, k, device="cuda", generator=g).to(dtype)
        bias = torch.randn(outputs, device="cuda", generator=g).to(dtype)
        wide = torch.full((tokens, outputs + 5), float("nan"), device="cuda", dtype=dtype)
        wide[:, 3:-2] = 2 * torch.randn(tokens, outputs, device="cuda", generator=g)
        residual = wide[:, 3:-2]
        plain = layer(x)
        for activation in (None, ("relu", "silu", "gelu", "gelu_tanh")[n % 4]):
            check(layer.linear(x, bias, activation, residual), layer, weights, x, bias, activation, residual)
        check(layer.linear(x, bias), layer, weights, x, bias, None, None)
        check(layer.linear(x, residual=residual), layer, weights, x, None, None, residual)
        check(layer.linear(x, activation="silu"), layer, weights, x, None, "silu", None)
        # nothing added changes nothing: the sums are the plain call's
        assert torch.equal(layer.linear(x, residual=torch.zeros_like(plain)), plain + 0)
        assert torch.equal(layer.linear(x), plain) and torch.equal(layer.linear(x, activation="none"), plain)
        packed = layer.run_packed(*native.pack(x), bias=bias, activation="gelu", residual=residual)
        assert torch.equal(packed, layer.linear(x, bias, "gelu", residual))
    assert layer.status()[0] == 0
    layer.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_activations_of_every_size(dtype):
    """Sums from -300 to 300 and the places where an activation bends, through the bias of a layer of zero weights."""
    v = torch.cat([torch.linspace(-300, 300, 601), torch.linspace(-6, 6, 1201), torch.tensor([0.0, -0.0, 1e-6, -1e-6, 6e4, -6e4])]).to(dtype)
    v = torch.cat([v, v.new_zeros(-v.numel() % 128)]).cuda()
    layer = native.DualLinear(torch.zeros(v.numel(), 128, dtype=dtype, device="cuda"), torch.arange(0, v.numel(), 5, device="cuda"))
    x = torch.ones(3, 128, dtype=dtype, device="cuda")
    for activation, function in REFERENCE.items():
        y = layer.linear(x, v, activation)
        want = function(v.double())
        tolerance = (torch.finfo(dtype).eps / 2 + 2.0 ** -19) * want.abs() + 2.0 ** -20 * v.double().abs().clamp(max=8) * torch.exp(-v.double().abs().clamp(max=20) / 2)
        assert bool(((y.double() - want).abs() <= tolerance + torch.finfo(dtype).smallest_normal).all()), activation
    nan = v.clone()
    nan[7], nan[8] = float("nan"), float("inf")
    y = layer.linear(x, nan, "relu")
    assert bool(y[:, 7].isnan().all()) and bool((y[:, 8] == float("inf")).all())
    layer.close()


def test_streams_and_graphs():
    layer, g = make(700, 896, 70, torch.bfloat16)
    for tokens in (5, 40):
        x, residual = (torch.randn(tokens, n, device="cuda", generator=g).bfloat16() for n in (896, 700))
        bias = torch.randn(700, device="cuda", generator=g).bfloat16()
        want = layer.linear(x, bias, "silu", residual)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = layer.linear(x, bias, "silu", residual)
        side.synchronize()
        assert torch.equal(got, want)
        buffer = torch.zeros_like(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = layer.linear(buffer, bias, "silu", residual)
        buffer.copy_(x)
        for _ in range(3):
            graph.replay()
            assert torch.equal(held, want)
    layer.close()


def test_refusals():
    layer, g = make(256, 256, 32, torch.bfloat16)
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    bias = y[0]
    for bad in (dict(bias=bias.float()), dict(bias=bias[:128]), dict(bias=bias.cpu()), dict(bias=y), dict(residual=y[:3]), dict(residual=y.half()),
                dict(residual=y.t().contiguous().t()), dict(activation="swish"), dict(bias=bias.clone().requires_grad_()),
                dict(residual=y.cpu())):
        with pytest.raises(ValueError):
            layer.linear(x, **bad)
        with pytest.raises(ValueError):
            layer.run_packed(*native.pack(x), **bad)
    for bad in (x.float(), x[:, :128], x.cpu(), x[0]):
        with pytest.raises(ValueError):
            layer.linear(bad, bias)
    assert layer.linear(x[:0], bias, residual=y[:0]).shape == (0, 256)
    explicit, _ = make(256, 256, 32, torch.bfloat16)
    explicit.low_id = explicit.high_id = 1
    with pytest.raises(ValueError, match="automatic schedule"):
        explicit.linear(x, bias)
    layer.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_decode_step(dtype):
    """The operators as a decoder block uses them: norm, qkv_proj with bias, cache, attention, o_proj and the residual, norm, gate_up_proj,
    SwiGLU and down_proj and the residual; each step against 64 bits from the step before, and the whole captured in a graph."""
    hidden, heads, kv_heads, dim, inter, seqs = 512, 8, 2, 64, 768, 5
    g = torch.Generator(device="cuda").manual_seed(3)

    def layer(outputs, k):
        weight = (0.05 * torch.randn(outputs, k, device="cuda", generator=g)).to(dtype)
        return native.DualLinear(weight, torch.arange(3, outputs, 10, device="cuda"))

    qkv, o_proj, gate_up, down = layer((heads + 2 * kv_heads) * dim, hidden), layer(hidden, heads * dim), layer(2 * inter, hidden), layer(hidden, inter)
    bias = torch.randn(qkv.outputs, device="cuda", generator=g).to(dtype)
    norms = [(1 + 0.2 * torch.randn(hidden, device="cuda", generator=g)).to(dtype) for _ in (0, 1)]
    cache = PagedCache.allocate(seqs * 8, 16, kv_heads, dim)
    table = torch.randperm(seqs * 8, device="cuda", generator=g).int().view(seqs, 8)
    past = torch.tensor([0, 1, 15, 16, 100], device="cuda")
    for position in range(100):   # what came before
        live = torch.nonzero(past > position).squeeze(1)
        slots = table[live, position // 16].long() * 16 + position % 16
        k, v = (torch.randn(live.numel(), kv_heads, dim, device="cuda", generator=g).to(dtype) for _ in (0, 1))
        cache.write(k, v, slots)
    slots = table[torch.arange(seqs, device="cuda"), past // 16].long() * 16 + past % 16
    lengths = (past + 1).int()
    x, residual = (torch.randn(seqs, hidden, device="cuda", generator=g).to(dtype) for _ in (0, 1))

    def step():
        q8, sf, h = producer.norm_pack(x, norms[0], 1e-6, residual)
        y = qkv.run_packed(q8, sf, bias=bias).unflatten(1, (-1, dim))
        cache.write(y[:, heads:heads + kv_heads], y[:, heads + kv_heads:], slots)
        a8, a_sf = cache.attention_pack(y[:, :heads], table, lengths)
        h1 = o_proj.run_packed(a8, a_sf, residual=h)
        n8, n_sf, _ = producer.norm_pack(h1, norms[1])
        z = gate_up.run_packed(n8, n_sf)
        d8, d_sf = producer.silu_pack(z)
        return h, y, a8, a_sf, h1, n8, n_sf, z, down.run_packed(d8, d_sf, residual=h1), d8, d_sf

    h, y, a8, a_sf, h1, n8, n_sf, z, out, d8, d_sf = step()
    def decoded(codes, scales):
        return torch.from_numpy(oracle.decode(codes.cpu().numpy(), scales.cpu().numpy(), codes.shape[1], fp4=False)).double().cuda()

    eps = torch.finfo(dtype).eps / 2
    for got, module, operand, extra in ((h1, o_proj, decoded(a8, a_sf), h), (z, gate_up, decoded(n8, n_sf), None), (out, down, decoded(d8, d_sf), h1)):
        weights = weights_of(module)
        want, size = operand @ weights.T, operand.abs() @ weights.abs().T
        if extra is not None:
            want, size = want + extra.double(), size + extra.double().abs()
        fp32 = (module.k * 2.0 ** -23 + 2.0 ** -21) * size
        assert bool(((got.double() - want).abs() <= eps * (want.abs() + fp32) + fp32).all())
    n = h1.double() / torch.sqrt(h1.double().square().mean(-1, keepdim=True) + 1e-6) * norms[1].double()
    assert bool(((decoded(n8, n_sf) - n).abs() <= 2.0 ** -4 * n.abs() + 2.0 ** -18 * n.abs() + 2.0 ** -10 * n.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(1) / 224).all())
    # against 64 bits: a 16-bit result of the same call is itself off by 2^-11 of the sum of its terms' sizes, which cancellation makes larger
    # than any multiple of the result
    want, _, size, score = attention_reference(cache, y[:, :heads], table, lengths, dim ** -0.5)
    check_packed(a8, a_sf, want.flatten(1), (bounds(dtype, want, size, score) - eps * want.abs()).flatten(1))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for t in held:
        t.zero_()
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, (h, y, a8, a_sf, h1, n8, n_sf, z, out, d8, d_sf)))
    for module in (qkv, o_proj, gate_up, down):
        module.close()


@pytest.mark.parametrize("activation, relative", [("silu", 2.0 ** -19), ("gelu", 2.0 ** -17), ("gelu_tanh", 2.0 ** -16)])
def test_small_results_of_activations(activation, relative):
    """Every bf16 value from -8 to -2^-10, where a result is up to 2^-47 of its argument: within the rounding of the exponent (an argument of up to 71
    of exp2, half a unit of fp32 in each of the steps to it), then rounded once.  Rounding keeps the order, so the bounds are rounded like the result."""
    v = torch.arange(0x3A80, 0x4101, device="cuda").to(torch.int16).view(torch.bfloat16).neg()
    v = torch.cat([v, v.new_zeros(-v.numel() % 128)])
    assert v.min() == -8 and v[0] == -2.0 ** -10
    layer = native.DualLinear(torch.zeros(v.numel(), 128, dtype=torch.bfloat16, device="cuda"), torch.arange(0, v.numel(), 5, device="cuda"))
    x = v.double()
    want = {"silu": x * torch.sigmoid(x), "gelu": 0.5 * x * torch.special.erfc(-x / math.sqrt(2)),
            "gelu_tanh": x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))}[activation]
    low, high = (want * (1 + relative)).bfloat16(), (want * (1 - relative)).bfloat16()
    for tokens in (3, 40):   # quantised in the launch, and ahead of it
        y = layer.linear(torch.ones(tokens, 128, dtype=torch.bfloat16, device="cuda"), v, activation)
        assert bool(((low <= y) & (y <= high)).all())
    layer.close()
