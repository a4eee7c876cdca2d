"""What stands between the linears, on the GPU, over the ways a call is spread over the device: attention of few long sequences and of many,
alike and ragged; the cache and norm of many rows; and every call by way of ctypes as by way of the host extension."""
import gc
import math

import pytest
import torch
from torch.autograd import forward_ad

from hygemm_vllm import native, producer
from hygemm_vllm.cache import PagedCache, page_bytes
from test_gpu_cache import TYPES, bounds, check_packed, filled, quantise, reference
from test_gpu_norm import FP32, check_codes, inputs, normed
from test_gpu_norm import reference as norm_reference

pytestmark = pytest.mark.gpu


def ragged(count, low, high, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(low, high + 1, (count,), generator=g).tolist()


PLANS = [
    # heads, kv_heads, head_dim, page, lengths, window
    (16, 8, 64, 16, ragged(2, 100, 180), 0),               # clusters of narrow blocks, or of wide ones
    (16, 8, 64, 16, ragged(3, 200, 400), 0),
    (8, 8, 128, 16, ragged(5, 300, 500), 0),
    (12, 6, 64, 32, ragged(11, 270, 700), 0),
    (14, 7, 128, 16, ragged(14, 260, 1000), 0),
    (16, 8, 64, 16, ragged(18, 260, 2000), 0),
    (8, 8, 64, 16, [32000], 0),                            # one sequence that fills the device
    (8, 4, 64, 16, ragged(16, 100, 9000), 0),              # few long ones, over a line of wide blocks
    (20, 2, 128, 32, ragged(30, 0, 5000), 0),
    (4, 2, 128, 16, [6000] * 70, 0),                       # as many as such blocks, alike
    (8, 4, 64, 16, ragged(20, 1, 20000), 6000),
    (28, 4, 128, 16, ragged(64, 10, 1000), 0),             # a line of blocks, three to an SM
    (8, 4, 64, 48, ragged(90, 0, 800), 0),
    (2, 1, 64, 16, [200000] + [3] * 159, 0),               # one sequence over hundreds of blocks
    (2, 1, 64, 16, [3] * 159 + [60000], 0),
    (4, 2, 128, 16, ragged(300, 0, 700), 0),               # four to an SM; more sequences than a block has threads
    (4, 4, 64, 64, ragged(413, 1, 900), 0),
    (20, 2, 64, 16, ragged(150, 1, 600), 0),               # two units of five heads and two more
    (8, 4, 64, 16, [700] * 160, 0),                        # alike: whole units
    (4, 4, 64, 16, ragged(444, 480, 500), 0),
    (8, 4, 128, 16, ragged(70, 1, 3000), 700),             # windows
    (4, 4, 64, 32, ragged(200, 1, 3000), 270),
    (2, 2, 64, 16, ragged(700, 0, 256), 0),                # short: whole units without a line
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", PLANS, ids=range(len(PLANS)))
def test_attention_plans(case, dtype):
    heads, kv_heads, dim, page, lengths, window = case
    cache, q, table, n = filled(len(lengths), heads, kv_heads, dim, page, lengths, dtype, seed=3)
    got, lse = cache.attention(q, table, n, window=window, lse=True)
    want, sums, size, score = reference(cache, q, table, n, dim ** -0.5, window)
    tolerance = bounds(dtype, want, size, score)
    assert bool(((got.double() - want).abs() <= tolerance).all())
    empty = n == 0
    assert bool((got[empty] == 0).all()) and bool((lse[empty] == -math.inf).all())
    assert bool(((lse.double() - sums)[~empty].abs() <= (2.0 ** -17 * score + 2.0 ** -18 + 2.0 ** -22 * sums.abs())[~empty]).all())
    assert torch.equal(got, cache.attention(q, table, n, window=window))
    codes, sf, packed_lse = cache.attention_pack(q, table, n, window=window, lse=True)
    assert torch.equal(packed_lse, lse)
    check_packed(codes, sf, want.flatten(1), (tolerance - torch.finfo(dtype).eps / 2 * want.abs()).flatten(1))


def test_workspaces():
    """Sums that cross blocks do not depend on what the workspace held, are kept apart in two graphs that run at once, and are the same in every replay."""
    lengths = ragged(64, 10, 1000)
    cache, q, table, n = filled(64, 28, 4, 128, 16, lengths, torch.bfloat16)
    half = n // 2
    first, second = cache.attention(q, table, n), cache.attention(q, table, half)
    gc.collect()
    for fill in (0x00, 0xFF, 0x3C):
        torch.cuda.synchronize()
        scratch = [torch.full((1 << 20,), fill, dtype=torch.uint8, device="cuda") for _ in range(8)]
        del scratch
        assert torch.equal(cache.attention(q, table, n), first)
    length = [n.clone(), half.clone()]
    graphs, outputs = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append([cache.attention(q, table, length[i]) for _ in range(3)])
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(30):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(outputs, (first, second)):
        assert all(torch.equal(t, want) for t in got)
    length[0].copy_(half)   # a replay reads what the lengths are then
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outputs[0][2], second)


def test_a_score_far_below_zero_counts():
    """One position, whose score is below -2^100: its weight is one all the same."""
    cache, q, table, n = filled(2, 8, 2, 64, 16, [1, 1], torch.bfloat16)
    got = cache.attention(q, table, n, scale=-(2.0 ** 110))
    again = cache.attention(q, table, n)
    assert torch.equal(got, again) and bool((got != 0).any())


def test_one_row_of_any_stride():
    """The stride of a single row says nothing."""
    cache, q, table, n = filled(1, 8, 2, 64, 16, [100], torch.float16)
    odd = torch.as_strided(q.contiguous(), q.shape, (3, 64, 1))
    assert torch.equal(cache.attention(odd, table, n), cache.attention(q, table, n))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_entries(dtype):
    """More than 2^15 heads of tokens in a call, and an odd number of tokens."""
    tokens, heads, dim, page = 8207, 4, 64, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    pages = 600
    cache = PagedCache(torch.full((pages, heads, page_bytes(page, dim)), 0xAA, dtype=torch.uint8, device="cuda"), page, dim)
    k, v = ((10 * torch.randn(tokens, heads, dim, device="cuda", generator=g)).to(dtype) for _ in (0, 1))
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens]
    slots[::7] = -1
    cache.write(k, v, slots)
    for got, x in zip(cache.read(slots, dtype), (k, v)):
        codes, e = quantise(x)
        want = (codes.double().unflatten(-1, (-1, 32)) * 2.0 ** e.double().unsqueeze(-1)).flatten(-2).to(torch.float32).to(dtype)
        want[slots < 0] = 0
        assert torch.equal(got, want)
    free = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    free[slots[slots >= 0]] = False
    untouched = cache.data[..., :2 * page * dim].view(pages, heads, 2, page, dim).permute(0, 3, 1, 2, 4).flatten(0, 1)[free]
    assert bool((untouched == 0xAA).all())


@pytest.mark.parametrize("case", [
    (768, 3584, torch.bfloat16, True, None, 1.0, False), (771, 1024, torch.float16, True, "channel", 1.0, True),
    (800, 1152, torch.float16, True, "token", 0.5, False), (1025, 8320, torch.bfloat16, False, "element", 1.0, True),
    (769, 18944, torch.bfloat16, True, None, 1.0, False), (1153, 8192, torch.bfloat16, True, "channel", 1.0, True),
    (770, 12288, torch.float16, True, None, 1.0, False), (1400, 7168, torch.bfloat16, False, "token", 2.0, False),
    (600, 16384, torch.bfloat16, True, "element", 1.0, True), (1600, 7296, torch.float16, False, None, 1.0, False)], ids=lambda c: f"{c[0]}x{c[1]}")
def test_norm_of_many_rows(case):
    operands = inputs(*case)
    q, sf, h = producer.norm_pack(eps=1e-6, **operands)
    x, weight = operands.pop("x"), operands.pop("weight")
    scale, post = operands.pop("scale"), operands.pop("post_weight")
    want, size = norm_reference(x, weight, 1e-6, operands["residual"], operands["gate"], scale, post, 1e-6)
    least = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert bool(((h.double() - want).abs() <= torch.finfo(x.dtype).eps / 2 * want.abs() + FP32 * size + least).all())
    check_codes(q, sf, normed(h, weight, 1e-6))


def test_calls_through_ctypes_are_the_same(monkeypatch):
    """What the host extension does not take, or where it is missing, goes through ctypes to the same kernels."""
    cache, q, table, n = filled(64, 28, 4, 128, 16, ragged(64, 10, 400), torch.bfloat16)
    operands = inputs(37, 896, torch.bfloat16, True, "element", 0.5, True)
    g = torch.Generator(device="cuda").manual_seed(1)
    weight = torch.randn(640, 896, device="cuda", generator=g).bfloat16()
    bias, residual = torch.randn(640, device="cuda", generator=g).bfloat16(), torch.randn(37, 640, device="cuda", generator=g).bfloat16()
    layer = native.DualLinear(weight, torch.arange(0, 640, 9, device="cuda"))
    slots = torch.tensor([5, -1, 40], device="cuda")

    def everything():
        results = [*producer.norm_pack(**operands), *producer.norm(**operands), layer.linear(operands["x"], bias, "gelu", residual),
                   cache.attention(q, table, n), *cache.attention(q, table, n, lse=True, window=100), *cache.attention_pack(q, table, n),
                   *cache.read(slots), *cache.read(slots, torch.float16)]
        cache.write(q[:3, 4:8], q[:3, 8:12], slots)
        results.append(cache.data.clone())
        cache.write(*cache.read(slots), slots)
        return results

    saved = cache.data.clone()
    fast = everything()
    cache.data.copy_(saved)
    monkeypatch.setattr(native, "_host", None)
    slow = everything()
    assert len(fast) == len(slow) and all(torch.equal(a, b) for a, b in zip(fast, slow))
    layer.close()


def test_no_gradient_is_asked_where_none_is_recorded():
    """Parameters need not be detached where gradients are off; where they are on, the calls say that they have none."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 896, device="cuda", generator=g).bfloat16()
    weight = torch.nn.Parameter(torch.randn(896, device="cuda", generator=g).bfloat16())
    layer = native.DualLinear(torch.randn(640, 896, device="cuda", generator=g).bfloat16(), torch.arange(0, 640, 9, device="cuda"))
    bias = torch.nn.Parameter(torch.randn(640, device="cuda", generator=g).bfloat16())
    for calls in (lambda: producer.norm(x, weight)[0], lambda: layer.linear(x, bias)):
        with pytest.raises(ValueError, match="gradient"):
            calls()
        for off in (torch.no_grad, torch.inference_mode):
            with off():
                got = calls()
            assert not got.requires_grad
    assert torch.equal(got, layer.linear(x, bias.detach()))
    layer.close()


@pytest.mark.parametrize("way", ["extension", "ctypes"])
def test_tangents_of_forward_mode_are_refused(way, monkeypatch):
    """The calls have no derivative: they say so for a tangent as for a recorded gradient, and take the tensor where forward mode is off."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x, weight = torch.randn(3, 896, device="cuda", generator=g).bfloat16(), torch.randn(896, device="cuda", generator=g).bfloat16()
    layer = native.DualLinear(torch.randn(640, 896, device="cuda", generator=g).bfloat16(), torch.arange(0, 640, 9, device="cuda"))
    bias, residual = torch.randn(640, device="cuda", generator=g).bfloat16(), torch.randn(3, 640, device="cuda", generator=g).bfloat16()
    cache, q, table, n = filled(3, 8, 2, 64, 16, [20, 3, 40], torch.bfloat16)
    kv, slots = q[:, :2].contiguous(), torch.tensor([1, 2, -1], device="cuda")
    layer.linear(x, bias)
    if way == "ctypes":
        monkeypatch.setattr(native, "_host", None)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda f=f, args=args: f(*args) for f, args in [
            (producer.norm, (dual(x), weight)), (producer.norm_pack, (x, dual(weight))), (producer.norm, (x, weight, 1e-6, dual(x))),
            (cache.attention, (dual(q), table, n)), (cache.attention_pack, (dual(q), table, n)), (cache.write, (dual(kv), kv, slots)),
            (cache.write, (kv, dual(kv), slots)), (layer.linear, (dual(x), bias)), (layer.linear, (x, dual(bias))),
            (layer.linear, (x, bias, "relu", dual(residual)))]]
        for call in calls:
            with pytest.raises(ValueError, match="gradient"):
                call()
            with forward_ad._set_fwd_grad_enabled(False):
                call()
            with torch.inference_mode():
                call()
        assert torch.equal(layer.linear(x, bias), layer.linear(x, bias.clone()))
    layer.close()
