"""The paged MXFP8 cache (`cache.PagedCache`) on the GPU: entries bit for bit, attention against 64-bit arithmetic."""
import math

import pytest
import torch

from hygemm_vllm.cache import PagedCache, page_bytes

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def quantise(v):
    """Codes and exponents of the last axis's groups of 32, from the definition: the smallest e with max|v| 2^-e <= 448, nearest codes."""
    groups = v.float().unflatten(-1, (-1, 32))
    amax = groups.abs().nan_to_num(0, torch.inf, 0).amax(-1)
    mantissa, e = torch.frexp(amax.clamp(max=3.4e38))
    e = torch.where(amax > 0, e - 9 + (mantissa > 0.875).int(), torch.zeros_like(e)).clamp(min=-127)
    e = torch.where(amax.isinf(), torch.full_like(e, 120), e)
    scaled = (groups.double() * 2.0 ** -e.double().unsqueeze(-1)).clamp(-448, 448).float()
    return scaled.to(torch.float8_e4m3fn).flatten(-2), e


def entry(cache, slot):
    """Codes [2, heads, head_dim] in the order of their elements, and scale bytes [2, heads, head_dim / 32], of one entry."""
    page, at = divmod(slot, cache.page_size)
    record, size, groups = cache.data[page], cache.page_size * cache.head_dim, cache.head_dim // 32
    d = torch.arange(cache.head_dim, device=record.device)
    order = (d % 32 // 4) * 4 * groups + d // 32 * 4 + d % 4
    codes = [record[:, i * size + at * cache.head_dim:][:, order] for i in (0, 1)]
    scales = [record[:, 2 * size + (2 * at + i) * groups:][:, :groups] for i in (0, 1)]
    return torch.stack(codes), torch.stack(scales)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head_dim, page, heads, tokens", [(128, 16, 4, 37), (64, 16, 3, 1), (64, 48, 1, 70), (128, 64, 8, 129), (128, 1024, 2, 5)])
def test_write_and_read(head_dim, page, heads, tokens, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    pages = -(-tokens // page) + 3
    cache = PagedCache(torch.full((pages, heads, page_bytes(page, head_dim)), 0xAA, dtype=torch.uint8, device="cuda"), page, head_dim)
    before = cache.data.clone()
    qkv = torch.randn(tokens, 5 * heads * head_dim, device="cuda", generator=g)
    qkv[:, ::9] *= 300
    qkv = qkv.to(dtype)
    k, v = (qkv[:, i * heads * head_dim:(i + 1) * heads * head_dim].unflatten(1, (heads, head_dim)) for i in (3, 4))
    k[0, 0, :32] = 0
    k[0, 0, 32:64] = torch.finfo(dtype).smallest_normal / 2      # a subnormal group
    v[0, 0, 5], v[0, 0, 40] = float("nan"), float("inf")
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens]
    written = slots.clone()
    if tokens > 4:
        slots[1], slots[2], slots[3] = -1, pages * page, 2 ** 40
    cache.write(k, v, slots)
    touched = torch.zeros(pages * page, dtype=torch.bool)
    for i, slot in enumerate(slots.tolist()):
        if not 0 <= slot < pages * page:
            continue
        touched[slot] = True
        codes, scales = entry(cache, slot)
        for kind, x in enumerate((k, v)):
            want, e = quantise(x[i])
            got, nan = codes[kind], want.float().isnan()
            assert torch.equal(got[~nan], want.view(torch.uint8)[~nan]) and bool(((got[nan] & 0x7F) == 0x7F).all())
            assert torch.equal(scales[kind].int() - 127, e.int())
    for slot in range(pages * page):
        if not touched[slot]:
            codes, scales = entry(cache, slot)
            assert bool((codes == 0xAA).all()) and bool((scales == 0xAA).all())
    # reading back: the values that codes and scales stand for, rounded once
    for to in TYPES:
        got = cache.read(slots, to)
        for kind, x in enumerate((k, v)):
            codes, e = quantise(x)
            want = (codes.double().unflatten(-1, (-1, 32)) * 2.0 ** e.double().unsqueeze(-1)).flatten(-2).to(torch.float32).to(to)
            want[(slots < 0) | (slots >= pages * page)] = 0
            assert torch.equal(got[kind].nan_to_num(7), want.nan_to_num(7))
    # the same slots again: an entry is replaced whole
    cache.write(v, k, slots)
    k2, v2 = cache.read(slots, dtype)
    cache.data.copy_(before)
    cache.write(k, v, slots)
    k1, v1 = cache.read(slots, dtype)
    assert torch.equal(k2.nan_to_num(7), v1.nan_to_num(7)) and torch.equal(v2.nan_to_num(7), k1.nan_to_num(7))
    assert written.shape == slots.shape


def dequantised(cache):
    """Keys and values [pages * page_size, heads, head_dim] in 64 bits."""
    p, n, groups = cache.page_size, cache.head_dim, cache.head_dim // 32
    size, out = p * n, []
    scales = cache.data[..., 2 * size:].unflatten(-1, (p, 2, groups)).double() - 127
    for i in (0, 1):
        codes = cache.data[..., i * size:(i + 1) * size].unflatten(-1, (p, 8, groups, 4)).transpose(-2, -3).flatten(-2)   # [.., p, groups, 32]
        value = codes.view(torch.float8_e4m3fn).double() * (2.0 ** scales[..., i, :]).unsqueeze(-1)
        out.append(value.flatten(-2).transpose(1, 2).flatten(0, 1))
    return out


def reference(cache, q, table, lengths, scale, window=0):
    """Outputs and log sums in 64 bits, and what the tolerances need: sum p |v| / sum p, and the largest scale sum |q| |k|."""
    keys, values = dequantised(cache)
    seqs, heads, dim = q.shape
    group = heads // cache.kv_heads
    out, size = (torch.zeros(seqs, heads, dim, dtype=torch.float64, device="cuda") for _ in (0, 1))
    lse, score = torch.full((seqs, heads), -math.inf, dtype=torch.float64, device="cuda"), torch.zeros(seqs, heads, dtype=torch.float64, device="cuda")
    for i in range(seqs):
        n = min(max(int(lengths[i]), 0), table.shape[1] * cache.page_size)
        position = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
        page = table[i][position // cache.page_size].long()
        there = (page >= 0) & (page < cache.pages)
        at = (page * cache.page_size + position % cache.page_size)[there]
        if not at.numel():
            continue
        k, v = keys[at].repeat_interleave(group, 1), values[at].repeat_interleave(group, 1)
        x = q[i].double()
        s = torch.einsum("hd,thd->ht", x, k) * scale
        p = torch.softmax(s, -1)
        out[i], size[i] = torch.einsum("ht,thd->hd", p, v), torch.einsum("ht,thd->hd", p, v.abs())
        lse[i] = torch.logsumexp(s, -1)
        score[i] = (torch.einsum("hd,thd->ht", x.abs(), k.abs()) * abs(scale)).amax(-1)
    return out, lse, size, score


def bounds(dtype, want, size, score):
    """A probability times the scale of its values is rounded to a half (2^-11 of it) in one product; a score is off by at most 64 roundings
    of 2^-23 of the sum of its terms' sizes, which changes each weight, and their sum, by as much; exponentials, sums and the joined
    parts by 2^-18.  One rounding to 16 bits comes last."""
    weight = 2.0 ** -11 + 2 * (2.0 ** -17 * score + 2.0 ** -18)
    return (torch.finfo(dtype).eps / 2) * want.abs() + weight.unsqueeze(-1) * size + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def filled(seqs, heads, kv_heads, dim, page, lengths, dtype, seed=0, spare=2, width=None, q_amplitude=2.0):
    """A cache of random entries, every byte outside the sequences 0xff (NaN codes, the largest scale), and shuffled pages; table entries
    behind a sequence's pages are no pages at all."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lengths]
    total = sum(need) + spare
    cache = PagedCache(torch.full((total, kv_heads, page_bytes(page, dim)), 0xFF, dtype=torch.uint8, device="cuda"), page, dim)
    order = torch.randperm(total, device="cuda", generator=g).int()
    table = torch.full((seqs, width or max(1, max(need))), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    at, slots = 0, []
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        position = torch.arange(max(lengths[i], 0), device="cuda")
        slots.append(order[at:at + n].long()[position // page] * page + position % page)
        at += n
    slots = torch.cat(slots) if slots else torch.empty(0, dtype=torch.int64, device="cuda")
    if slots.numel():
        k = torch.randn(slots.numel(), kv_heads, dim, device="cuda", generator=g)
        k[..., ::13] *= 5
        cache.write(k.to(dtype), torch.randn(slots.numel(), kv_heads, dim, device="cuda", generator=g).to(dtype), slots)
    qkv = (q_amplitude * torch.randn(seqs, heads + 2 * kv_heads, dim, device="cuda", generator=g)).to(dtype)
    return cache, qkv[:, :heads], table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


CASES = [
    # heads, kv_heads, head_dim, page, lengths, window
    (28, 4, 128, 16, [1], 0),
    (28, 4, 128, 16, [1000], 0),
    (4, 4, 64, 16, [0, 1, 15, 16, 17, 31, 32, 33], 0),
    (8, 1, 128, 16, [0, 0, 5], 0),
    (32, 8, 128, 32, [31, 32, 33, 700, 1], 0),
    (5, 1, 64, 48, [47, 48, 49, 300], 0),
    (12, 1, 128, 64, [129, 2049, 7], 0),
    (34, 2, 64, 16, [260, 257, 255], 0),
    (7, 1, 128, 1024, [1023, 1024, 1025], 0),
    (28, 4, 128, 16, [9000, 3, 4097], 0),
    (16, 2, 64, 16, [20000], 0),
    (2, 2, 128, 16, [257] * 70, 0),
    (8, 2, 128, 16, [1, 15, 16, 100, 5000], 16),
    (8, 2, 64, 32, [1, 15, 16, 100, 5000], 1),
    (6, 3, 128, 16, [3000, 700, 8], 1000),
    (8, 8, 128, 16, [40, 3000], 3000),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
def test_attention(case, dtype):
    heads, kv_heads, dim, page, lengths, window = case
    cache, q, table, n = filled(len(lengths), heads, kv_heads, dim, page, lengths, dtype)
    got, lse = cache.attention(q, table, n, window=window, lse=True)
    want, sums, size, score = reference(cache, q, table, n, dim ** -0.5, window)
    assert got.shape == q.shape and got.dtype == dtype
    assert bool(((got.double() - want).abs() <= bounds(dtype, want, size, score)).all())
    empty = n == 0
    assert torch.equal(got[empty], torch.zeros_like(got[empty])) and bool((lse[empty] == -math.inf).all())
    assert bool(((lse.double() - sums)[~empty].abs() <= (2.0 ** -17 * score + 2.0 ** -18 + 2.0 ** -22 * sums.abs())[~empty]).all())
    assert torch.equal(got, cache.attention(q, table, n, window=window)), "the same call gives the same bits"
    if heads * dim % 128 == 0:
        codes, sf, packed_lse = cache.attention_pack(q, table, n, window=window, lse=True)
        assert torch.equal(packed_lse, lse)
        check_packed(codes, sf, want.flatten(1), (bounds(dtype, want, size, score) - torch.finfo(dtype).eps / 2 * want.abs()).flatten(1))


def check_packed(codes, sf, want, off):
    """`want` in 64 bits, fp32 results at most `off` from it, then quantised: the scale fits the largest, a code is half a step off."""
    rows, k = want.shape
    atoms = sf.view(-1, k // 128, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, k // 32)
    assert codes.shape == (rows, k) and bool((atoms[rows:] == 127).all())
    e = atoms[:rows].double() - 127
    amax, slack = want.unflatten(-1, (-1, 32)).abs().amax(-1), off.unflatten(-1, (-1, 32)).amax(-1)
    live = amax > 0
    assert bool((amax - slack <= 448 * 2.0 ** e)[live].all()) and bool((amax + slack > 224 * 2.0 ** e)[live].all())
    value = (codes.view(torch.float8_e4m3fn).double().unflatten(-1, (-1, 32)) * (2.0 ** e).unsqueeze(-1)).flatten(-2)
    step = 2.0 ** -10 * (2.0 ** e).repeat_interleave(32, -1)
    assert bool(((value - want).abs() <= off + 2.0 ** -4 * (want.abs() + off) + step).all())
    assert bool((e[~live] == 0).all()) and bool((value[want == 0] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_pages_that_are_not_there(dtype):
    """Positions of a page number outside the cache are left out, wherever in a sequence; a row may lose all of them."""
    cache, q, table, n = filled(3, 8, 2, 128, 16, [100, 600, 40], dtype)
    table[0, 2], table[1, 0], table[1, 20], table[1, 37] = -1, cache.pages, 2 ** 31 - 1, -2 ** 31
    table[2] = -1
    got, lse = cache.attention(q, table, n, lse=True)
    want, sums, size, score = reference(cache, q, table, n, 128 ** -0.5)
    assert bool(((got.double() - want).abs() <= bounds(dtype, want, size, score)).all())
    assert bool((got[2] == 0).all()) and bool((lse[2] == -math.inf).all())


def test_lengths_outside_the_table():
    cache, q, table, n = filled(3, 8, 2, 128, 16, [32, 32, 32], torch.bfloat16)
    beyond = torch.tensor([1000, 32, -5], dtype=torch.int32, device="cuda")
    got = cache.attention(q, table, beyond)
    assert torch.equal(got[:2], cache.attention(q, table, n)[:2]) and bool((got[2] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_and_scales_of_every_size(dtype):
    """Scores in the hundreds, rising and falling; values whose scales lie 2^20 apart, the largest last, first or under a small weight."""
    g = torch.Generator(device="cuda").manual_seed(5)
    for order in ("rising", "falling", "shuffled"):
        cache, q, table, n = filled(2, 8, 2, 128, 16, [333, 1500], dtype, seed=9, q_amplitude=12.0)
        slots = torch.cat([table[i].long()[torch.arange(m, device="cuda") // 16] * 16 + torch.arange(m, device="cuda") % 16 for i, m in enumerate((333, 1500))])
        exponent = torch.linspace(-10, 10, slots.numel(), device="cuda").round()
        if order == "falling":
            exponent = exponent.flip(0)
        if order == "shuffled":
            exponent = exponent[torch.randperm(slots.numel(), device="cuda", generator=g)]
        k, v = (torch.randn(slots.numel(), 2, 128, device="cuda", generator=g) for _ in (0, 1))
        cache.write(k.to(dtype), (v * (2.0 ** exponent).view(-1, 1, 1)).to(dtype), slots)
        got = cache.attention(q, table, n)
        want, _, size, score = reference(cache, q, table, n, 128 ** -0.5)
        assert bool(((got.double() - want).abs() <= bounds(dtype, want, size, score)).all()), order
        assert bool(got.isfinite().all())


GROUPS_OF_VALUES = [
    # types, exponent of each scale group's values, tokens (of 48) whose values are zeros, of which groups
    (TYPES, [-13, -13, -13, None], "none", ()),                 # a head padded with zeros: 2^-13 is 1.2e-4
    (TYPES, [None, -8, None, -13], "none", ()),
    ([torch.bfloat16], [-20, -20, -20, None], "none", ()),
    ([torch.bfloat16], [-80, None, -60, -40], "none", ()),
    (TYPES, [10, -2, -8, -13], "none", ()),
    ([torch.bfloat16], [30, 10, -10, -30], "none", ()),
    ([torch.bfloat16], [0, -40, -80, 40], "none", ()),
    ([torch.bfloat16], [100, -90, 60, 118], "none", ()),        # up to 2^120: sums stay in range
    (TYPES, [-13, -13, -13, -13], "every third", (0, 1, 2, 3)),  # zeros between small values
    ([torch.bfloat16], [-20, 0, -40, -20], "every third", (0, 1, 2)),
    ([torch.bfloat16], [-20, -20, 0, -40], "the first", (0, 3)),  # zeros only, then small values
    ([torch.bfloat16], [-20, -20, 8, -40], "the last", (0, 2, 3)),
    ([torch.bfloat16], [-20, 0, -30, -40], "but one", (0, 2)),   # zeros only, up to one
]


@pytest.mark.parametrize("heads, kv_heads, dim, lengths", [(8, 2, 128, [333, 1500, 17]), (4, 2, 64, [1500, 40]), (28, 4, 128, [300] * 64), (3, 1, 64, [700] * 160)])
@pytest.mark.parametrize("case", range(len(GROUPS_OF_VALUES)))
def test_values_of_groups_of_every_size(case, heads, kv_heads, dim, lengths):
    """The scale groups of a head differ by any factor, or are zeros, in all entries or in some: each output is as near as its own group's values allow.
    Sixteen bits add half a step; quantised outputs are held to fp32's error and the rounding of a weight alone."""
    types, exponents, where, zero_groups = GROUPS_OF_VALUES[case]
    for dtype in types:
        cache, q, table, n = filled(len(lengths), heads, kv_heads, dim, 16, lengths, dtype, seed=case)
        g = torch.Generator(device="cuda").manual_seed(case + 1)
        position = torch.cat([torch.arange(m, device="cuda") for m in lengths])
        slots = torch.cat([table[i].long()[torch.arange(m, device="cuda") // 16] * 16 + torch.arange(m, device="cuda") % 16 for i, m in enumerate(lengths)])
        k, v = (torch.randn(slots.numel(), kv_heads, dim, device="cuda", generator=g) for _ in (0, 1))
        zero = {"none": position < 0, "every third": position % 3 == 0, "the first": position < 210, "the last": position >= 20, "but one": position != 14}[where]
        for group in range(dim // 32):
            part = v[..., 32 * group:32 * group + 32]
            part.mul_(0.0 if exponents[group] is None else 2.0 ** exponents[group])
            if group in zero_groups:
                part[zero] = 0
        cache.write(k.to(dtype), v.to(dtype), slots)
        got, lse = cache.attention(q, table, n, lse=True)
        want, sums, size, score = reference(cache, q, table, n, dim ** -0.5)
        assert bool(((got.double() - want).abs() <= bounds(dtype, want, size, score)).all())
        assert bool(((lse.double() - sums).abs() <= 2.0 ** -17 * score + 2.0 ** -18 + 2.0 ** -22 * sums.abs()).all())
        if heads * dim % 128 == 0:
            codes, sf, packed_lse = cache.attention_pack(q, table, n, lse=True)
            assert torch.equal(packed_lse, lse)
            weight = 2.0 ** -11 + 2 * (2.0 ** -17 * score + 2.0 ** -18)
            check_packed(codes, sf, want.flatten(1), (weight.unsqueeze(-1) * size).flatten(1))


@pytest.mark.parametrize("amplitude", [0.0, 2.0 ** -100, 2.0 ** 60])
def test_queries_of_every_size(amplitude):
    """bf16 queries beyond the range of a half: the scores are what they are, with a scale that brings them back."""
    cache, q, table, n = filled(2, 8, 2, 64, 16, [50, 300], torch.bfloat16, q_amplitude=1.0)
    scale = 64 ** -0.5 / (amplitude or 1.0)
    got = cache.attention((q.float() * amplitude).bfloat16(), table, n, scale=scale)
    want, _, size, score = reference(cache, (q.float() * amplitude).bfloat16(), table, n, scale)
    assert bool(((got.double() - want).abs() <= bounds(torch.bfloat16, want, size, score)).all())


def test_nan_and_infinity_stay_in_their_rows():
    cache, q, table, n = filled(3, 8, 2, 128, 16, [100, 100, 100], torch.bfloat16)
    good = cache.attention(q, table, n)
    q = q.clone()
    q[1, 2, 7] = float("nan")
    got = cache.attention(q, table, n)
    assert bool(got[1, 2].isnan().all()) and torch.equal(got[[0, 2]], good[[0, 2]])
    slot = table[2, 3].long() * 16 + 5
    k, v = cache.read(slot.view(1))
    v[0, 1, 9] = float("nan")
    cache.write(k, v, slot.view(1))
    got = cache.attention(q, table, n)
    assert bool(got[2, 4:, 9].isnan().all()) and not bool(got[2, :4].isnan().any()) and torch.equal(got[0], good[0])
    assert not bool(got[2, 4:, :9].isnan().any())


def test_strided_operands():
    cache, q, table, n = filled(5, 8, 2, 128, 16, [100, 37, 1, 0, 512], torch.float16)
    wide = torch.full((5, table.shape[1] + 3), -7, dtype=torch.int32, device="cuda")
    wide[:, :-3] = table
    assert q.stride(0) != 8 * 128
    assert torch.equal(cache.attention(q, wide[:, :-3], n), cache.attention(q.contiguous(), table, n))


def test_streams_and_graphs():
    """Captured calls read the lengths, tables and entries of their replay; two graphs keep workspaces of their own."""
    cache, q, table, n = filled(3, 8, 2, 128, 16, [3000, 900, 20], torch.bfloat16)
    first, second = cache.attention(q, table, n), cache.attention(q, table, n // 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attention(q, table, n)
    side.synchronize()
    assert torch.equal(got, first)
    lengths = [n.clone(), n.clone()]
    graphs, outputs = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append(cache.attention(q, table, lengths[i]))
        graphs.append(graph)
    lengths[1].copy_(n // 2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outputs[0], first) and torch.equal(outputs[1], second)


def test_write_then_attention_without_a_wait():
    """A decode loop: each step writes an entry and reads it in the next launch."""
    cache, q, table, n = filled(4, 8, 2, 128, 16, [64, 64, 64, 64], torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(2)
    steps = []
    for step in range(60):
        k, v = (torch.randn(4, 2, 128, device="cuda", generator=g).bfloat16() for _ in (0, 1))
        place = torch.full((4,), step, device="cuda")
        slots = table.gather(1, (place // 16).unsqueeze(1)).squeeze(1).long() * 16 + place % 16
        cache.write(k, v, slots)
        length = (place + 1).int()
        steps.append((length, cache.attention(q, table, length)))
    for length, got in steps:
        assert torch.equal(got, cache.attention(q, table, length))


def test_nothing_to_do():
    cache = PagedCache.allocate(2, 16, 2, 64)
    empty = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    table, n = torch.empty(0, 3, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    assert cache.attention(empty, table, n).shape == (0, 4, 64)
    codes, sf = cache.attention_pack(empty, table, n)
    assert codes.shape == (0, 256) and sf.numel() == 0
    cache.write(empty[:, :2], empty[:, :2], torch.empty(0, dtype=torch.int64, device="cuda"))
    assert cache.read(torch.empty(0, dtype=torch.int64, device="cuda"))[0].shape == (0, 2, 64)
    one = torch.ones(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    none = cache.attention(one, torch.empty(1, 0, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"))
    assert bool((none == 0).all())


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes: entries at its end."""
    pages, page, heads, dim = 17000, 256, 4, 128
    cache = PagedCache(torch.empty(pages, heads, page_bytes(page, dim), dtype=torch.uint8, device="cuda"), page, dim)
    assert cache.data.numel() > 2 ** 32
    g = torch.Generator(device="cuda").manual_seed(4)
    table = torch.tensor([[pages - 1, pages - 2], [pages - 3, pages - 4]], dtype=torch.int32, device="cuda")
    position = torch.arange(400, device="cuda")
    slots = torch.cat([table[i].long()[position // page] * page + position % page for i in (0, 1)])
    k, v = (torch.randn(800, heads, dim, device="cuda", generator=g).bfloat16() for _ in (0, 1))
    cache.write(k, v, slots)
    small = PagedCache.allocate(4, page, heads, dim)
    cache_pages = torch.tensor([[3, 2], [1, 0]], dtype=torch.int32, device="cuda")
    small.write(k, v, torch.cat([cache_pages[i].long()[position // page] * page + position % page for i in (0, 1)]))
    assert torch.equal(cache.read(slots)[0], small.read(torch.cat([cache_pages[i].long()[position // page] * page + position % page for i in (0, 1)]))[0])
    q = torch.randn(2, 8, dim, device="cuda", generator=g).bfloat16()
    n = torch.tensor([400, 399], dtype=torch.int32, device="cuda")
    assert torch.equal(cache.attention(q, table, n), small.attention(q, cache_pages, n))


def test_refusals():
    cache = PagedCache.allocate(4, 16, 2, 64)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    table, n = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    kv = q[:, :2]
    for bad in (q.float(), q[:, :3], q[..., :32], q[0], q.cpu(), torch.zeros(2, 64, 4, dtype=torch.bfloat16, device="cuda").transpose(1, 2)):
        with pytest.raises(ValueError):
            cache.attention(bad, table, n)
    for bad in (table.long(), table[:1], table.cpu(), table[0]):
        with pytest.raises(ValueError, match="page table"):
            cache.attention(q, bad, n)
    for bad in (n.long(), n[:1], n.cpu(), n.view(2, 1)):
        with pytest.raises(ValueError, match="lengths"):
            cache.attention(q, table, bad)
    with pytest.raises(ValueError, match="window"):
        cache.attention(q, table, n, window=-1)
    with pytest.raises(ValueError, match="divisible by 128"):
        PagedCache.allocate(4, 16, 1, 64).attention_pack(q[:, :3], table, n)
    with pytest.raises(ValueError, match="gradient"):
        cache.attention(q.clone().requires_grad_(), table, n)
    for k, v, s in ((kv.float(), kv.float(), slots), (kv, kv.half(), slots), (kv[:1], kv[:1], slots), (q, q, slots), (kv, kv, slots.int()),
                    (kv, kv, slots.cpu()), (kv.transpose(0, 1).contiguous().transpose(0, 1)[..., ::2], kv[..., ::2], slots),
                    (kv, kv, torch.zeros(4, dtype=torch.int64, device="cuda")[::2])):
        with pytest.raises(ValueError):
            cache.write(k, v, s)
    with pytest.raises(ValueError):
        cache.read(slots, torch.float32)
    data = cache.data
    for bad, page, dim in ((data, 16, 128), (data, 8, 64), (data, 24, 64), (data.cpu(), 16, 64), (data.int(), 16, 64), (data[:, :, :-1], 16, 64),
                           (data[:0], 16, 64), (data, 16, 96), (data, 0, 64), (data, 2048, 64)):
        with pytest.raises(ValueError):
            PagedCache(bad, page, dim)
