"""Norm with residual and quantisation (`producer.norm_pack`, `producer.norm`) on the GPU against 64-bit arithmetic.

Tolerances.  h is rounded once to 16 bits (half a step, eps / 2) behind at most six fp32 operations on its terms (each
2^-24 of a partial result, at most the sum of the terms' sizes).  n is computed from h by fp32: a sum of K squares, rsqrtf (2 units) and
two products, under K 2^-24 / 2 + 2^-21 of the value, K at most 32768; sums are added in parts, so 2^-18 covers them.  An E4M3
code is half a step off: 2^-4 of the value, or 2^-10 of the scale below 2^-6 of it.
"""
import pytest
import torch

import oracle
from hygemm_vllm import native, producer

pytestmark = pytest.mark.gpu
FP32 = 2.0 ** -18


def logical_scales(sf, rows, k):
    """Exponents [rows, k / 32] out of the atoms; every padding byte is 0x7f."""
    atoms = sf.cpu().view(-1, k // 128, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, k // 32)
    assert bool((atoms[rows:] == 127).all())
    return atoms[:rows].int() - 127


def reference(x, weight, eps, residual, gate, scale, post, post_eps):
    """h in 64 bits, and the sizes of its terms."""
    y = x.double()
    if post is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + post_eps) * post.double()
    if gate is not None:
        y = y * gate.double()
    y = y * scale
    size = y.abs()
    if residual is not None:
        y, size = y + residual.double(), size + residual.double().abs()
    return y, size


def normed(h, weight, eps):
    h = h.double()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double()


def check_codes(q, sf, n):
    rows, k = n.shape
    e = logical_scales(sf, rows, k).cuda().double()
    amax = n.unflatten(-1, (-1, 32)).abs().amax(-1)
    scaled = amax * 2.0 ** -e
    live = amax > 2.0 ** -118
    assert bool((scaled[live] <= 448 * (1 + FP32)).all()) and bool((scaled[live] > 224 * (1 - FP32)).all())
    assert bool((e[amax == 0] == 0).all())
    value = q.view(torch.float8_e4m3fn).double().unflatten(-1, (-1, 32)) * (2.0 ** e).unsqueeze(-1)
    n = n.unflatten(-1, (-1, 32))
    tolerance = (2.0 ** -4 + FP32) * n.abs() + 2.0 ** -10 * (2.0 ** e).unsqueeze(-1)
    assert bool(((value - n).abs() <= tolerance).all())


CASES = [
    # rows, k, dtype, residual, gate, scale, post
    (1, 128, torch.bfloat16, True, None, 1.0, False),
    (1, 3584, torch.bfloat16, True, None, 1.0, False),
    (3, 384, torch.float16, False, None, 1.0, False),
    (5, 2432, torch.float16, True, "channel", 0.25, True),
    (129, 896, torch.bfloat16, True, "element", 1.0, True),
    (128, 1152, torch.float16, True, "token", -2.5, False),
    (37, 8192, torch.bfloat16, False, None, 1.0, True),
    (2, 8320, torch.bfloat16, True, None, 1.0, False),
    (3, 18944, torch.float16, True, "channel", 1.0, True),
    (2, 32768, torch.bfloat16, True, "element", 0.5, True),
    (300, 4096, torch.bfloat16, True, None, 1.0, False),
    (2, 640, torch.bfloat16, False, "token", 1.0, False),
]


def inputs(rows, k, dtype, residual, gate, scale, post, strided=False, seed=7):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    def matrix(amplitude):
        wide = torch.full((rows, k + 24), float("nan"), device="cuda", dtype=dtype) if strided else None
        x = (amplitude * randn(rows, k)).to(dtype)
        if wide is None:
            return x
        wide[:, 8:8 + k] = x
        return wide[:, 8:8 + k]

    x = matrix(1)
    x[:, ::17] *= 20
    shape = {None: None, "channel": (k,), "element": (rows, k), "token": (rows, 1)}[gate]
    return dict(x=x, weight=(1 + 0.3 * randn(k)).to(dtype), residual=matrix(4) if residual else None,
                gate=None if shape is None else (matrix(1) if gate == "element" else randn(*shape).to(dtype)), scale=scale,
                post_weight=(1 + 0.3 * randn(k)).to(dtype) if post else None)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}")
def test_norm(case, strided):
    rows, k, dtype = case[:3]
    a = inputs(*case, strided=strided)
    eps, post_eps = 1e-5, 1e-3
    q, sf, h = producer.norm_pack(a["x"], a["weight"], eps, a["residual"], gate=a["gate"], scale=a["scale"],
                                  post_weight=a["post_weight"], post_eps=post_eps)
    n, h2 = producer.norm(a["x"], a["weight"], eps, a["residual"], gate=a["gate"], scale=a["scale"],
                          post_weight=a["post_weight"], post_eps=post_eps)
    assert q.shape == (rows, k) and q.dtype == torch.uint8 and sf.numel() == native.scale_size(rows, k)
    assert h.dtype == n.dtype == dtype and torch.equal(h, h2)
    want, size = reference(a["x"], a["weight"], eps, a["residual"], a["gate"], a["scale"], a["post_weight"], post_eps)
    step = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).smallest_normal * step * 2
    assert bool(((h.double() - want).abs() <= step * want.abs() + FP32 * size + least).all())
    exact = normed(h, a["weight"], eps)
    assert bool(((n.double() - exact).abs() <= (step + FP32) * exact.abs() + least).all())
    check_codes(q, sf, exact)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_unchanged_stream_is_the_input(dtype):
    a = inputs(4, 256, dtype, False, None, 1.0, False)
    q, sf, h = producer.norm_pack(a["x"], a["weight"])
    assert h is a["x"]
    assert producer.norm(a["x"], a["weight"])[1] is a["x"]


def test_quantisation_is_packs():
    """With rows whose root mean square and weights are one, n is h up to an fp32 unit: codes are native.pack's of h almost everywhere."""
    g = torch.Generator(device="cuda").manual_seed(3)
    signs = torch.randint(0, 2, (70, 512), device="cuda", generator=g) * 2 - 1
    h = signs.bfloat16()                                    # mean square exactly one
    weight = torch.randn(512, device="cuda", generator=g).bfloat16()
    q, sf, _ = producer.norm_pack(h, weight, 0.0)
    want_q, want_sf = native.pack(h * weight)               # exact products: rsqrt(1) is 1
    assert torch.equal(q, want_q) and torch.equal(sf, want_sf)


def test_no_rows_and_extremes():
    empty = torch.empty((0, 256), dtype=torch.bfloat16, device="cuda")
    weight = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    q, sf, h = producer.norm_pack(empty, weight, residual=empty)
    assert q.shape == h.shape == (0, 256) and sf.numel() == 0
    x = torch.zeros((4, 256), dtype=torch.bfloat16, device="cuda")
    x[1, 3], x[2, 5], x[3] = float("nan"), float("inf"), 2.0 ** -120
    q, sf, _ = producer.norm_pack(x, weight, 1e-6)
    assert bool((q[0] == 0).all()) and bool((logical_scales(sf, 4, 256)[0] == 0).all())
    values = q.view(torch.float8_e4m3fn).float()
    assert bool(values[1].isnan().all())                    # the row's mean square is NaN
    n, _ = producer.norm(x, weight, 1e-6)
    assert bool(n[0].eq(0).all()) and bool(n[1].isnan().all()) and bool(n[2, 5].isnan()) and bool((n[2, :5] == 0).all())
    assert bool(((n[3].double() / (2.0 ** -120 * 1000) - 1).abs() <= 2.0 ** -9 + FP32).all())


def test_streams_and_graphs():
    a = inputs(19, 640, torch.bfloat16, True, "channel", 0.5, True)
    call = lambda x: producer.norm_pack(x, a["weight"], 1e-6, a["residual"], gate=a["gate"], scale=0.5, post_weight=a["post_weight"])  # noqa: E731
    want = [t.clone() for t in call(a["x"])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(a["x"])
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    buffer = torch.zeros_like(a["x"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(buffer)
    for _ in range(2):
        buffer.copy_(a["x"])
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(held, want))
        buffer.zero_()
        graph.replay()
        assert not torch.equal(held[0], want[0])


def test_layer_on_its_output():
    """norm_pack feeds run_packed as pack does."""
    a = inputs(6, 512, torch.bfloat16, True, None, 1.0, False)
    g = torch.Generator(device="cuda").manual_seed(1)
    layer = native.DualLinear((0.02 * torch.randn(384, 512, device="cuda", generator=g)).bfloat16(),
                              torch.arange(0, 384, 10, device="cuda"))
    q, sf, h = producer.norm_pack(a["x"], a["weight"], 1e-6, a["residual"])
    y = layer.run_packed(q, sf)
    x = oracle.decode(q.cpu().numpy(), sf.cpu().numpy(), 512, fp4=False)
    w = torch.empty(384, 512, dtype=torch.float64)
    w[layer.lo.long().cpu()] = torch.from_numpy(oracle.decode(layer.w4.cpu().numpy(), layer.sf4.cpu().numpy(), 512, fp4=True)).double()
    w[layer.hi.long().cpu()] = torch.from_numpy(oracle.decode(layer.w8.cpu().numpy(), layer.sf8.cpu().numpy(), 512, fp4=False)).double()
    want = torch.from_numpy(x).double() @ w.T
    size = torch.from_numpy(x).double().abs() @ w.T.abs()
    assert bool(((y.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 512 * 2.0 ** -22 * size).all())
    layer.close()


@pytest.mark.parametrize("change, message", [
    (dict(x=torch.zeros(2, 250, dtype=torch.bfloat16)), "divisible"),
    (dict(x=torch.zeros(2, 256)), "FP16/BF16"),
    (dict(x=torch.zeros(512, dtype=torch.bfloat16)), "FP16/BF16"),
    (dict(x=torch.zeros(256, 2, dtype=torch.bfloat16).t()), "aligned"),
    (dict(residual=torch.zeros(3, 256, dtype=torch.bfloat16)), "residual"),
    (dict(residual=torch.zeros(2, 256, dtype=torch.float16)), "residual"),
    (dict(weight=torch.zeros(128, dtype=torch.bfloat16)), "weights"),
    (dict(post_weight=torch.zeros(256)), "weights"),
    (dict(gate=torch.zeros(2, 128, dtype=torch.bfloat16)), "gate"),
    (dict(gate=torch.zeros(256, 2, dtype=torch.bfloat16).t()), "gate"),
], ids=range(10))
def test_refusals(change, message):
    a = dict(x=torch.zeros(2, 256, dtype=torch.bfloat16), weight=torch.zeros(256, dtype=torch.bfloat16)) | change
    a = {name: t.cuda() for name, t in a.items()}
    x, weight = a.pop("x"), a.pop("weight")
    if message == "divisible":
        weight = torch.zeros(250, dtype=torch.bfloat16, device="cuda")
    for call in (producer.norm_pack, producer.norm):
        with pytest.raises(ValueError, match=message):
            call(x, weight, 1e-6, **a)
    with pytest.raises(ValueError, match="gradient"):
        producer.norm(torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda").requires_grad_(), torch.zeros(256, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("way", ["extension", "ctypes"])
def test_a_scale_that_rounds_to_one(way, monkeypatch):
    """The kernel takes the scale in fp32: one that is 1 there leaves the stream as it is, whichever way the call goes."""
    a = inputs(4, 256, torch.bfloat16, False, None, 1.0, False)
    producer.norm(a["x"], a["weight"])
    if way == "ctypes":
        monkeypatch.setattr(native, "_host", None)
    for scale in (1 + 1e-9, 2 ** .5 * .5 ** .5, 1 - 2.0 ** -26):
        held = torch.full((4, 256), float("nan"), dtype=torch.bfloat16, device="cuda")
        del held   # what an allocation finds there
        assert producer.norm(a["x"], a["weight"], scale=scale)[1] is a["x"]
        assert producer.norm_pack(a["x"], a["weight"], scale=scale)[2] is a["x"]
    n, h = producer.norm(a["x"], a["weight"], scale=1 + 2.0 ** -22)   # not 1 in fp32, and nothing for bf16
    assert h is not a["x"] and torch.equal(h, a["x"])
