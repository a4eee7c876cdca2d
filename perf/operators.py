"""The operators that stand between the hybrid linears of a decoder block, as cases that can be timed and compared.

Four kinds of pass:

* "norm":      residual add (with a gate, a residual scale and a norm of the block's output in front, where the model has
               them), RMS norm, and MXFP8 quantisation of the normalised rows: what stands before qkv_proj and gate_up_proj
               (`producer.norm_pack`), and with 16-bit rows before an unquantised lm_head (`producer.norm`).
* "write" and "read":  new keys and values quantised to MXFP8 into the pages of a cache (`PagedCache.write`), and entries
               read back in 16 bits (`PagedCache.read`).
* "attention": one new token a sequence over that cache (`PagedCache.attention`), or with its output as the MXFP8 input
               of o_proj (`PagedCache.attention_pack`).
* "linear":    a hybrid MXFP4/MXFP8 linear with bias, activation and residual in its epilogue (`DualLinear.linear`).

The plain form is written in elementary torch operations, in 32 bits, rounded once at the end.  MXFP8 means E4M3 codes with
one E8M0 scale 2^e per 32 values, e the smallest exponent with max|v| 2^-e <= 448.

Layout of a cache, uint8 [pages, kv_heads, page_bytes], per page and head: key codes [page_size][head_dim], value codes
[page_size][head_dim], scales [page_size][keys, values][head_dim / 32].  A token's codes lie as [8][head_dim / 32][4]: element
d = 32 g + 4 x + i at (x, g, i).
"""
import functools
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_MOST_CACHED = 4 * 32768 * 4 * 128   # elements of the keys of a drawn cache at most


@functools.cache
def _framework():
    path = os.path.join(os.getcwd(), "comp2029-hybridgemm_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from hygemm_vllm import cache, native, producer
    return cache, native, producer


def _norm(name, rows, k, dtype="bf16", residual=True, post=False, gate="none", scale=1.0, packed=True):
    return {"name": name, "kind": "norm", "rows": rows, "k": k, "dtype": dtype, "residual": residual, "post": post,
            "gate": gate, "scale": scale, "packed": packed}


def _cache(name, kind, tokens, kv_heads, head_dim, page, pages, dtype="bf16", absent=0):
    return {"name": name, "kind": kind, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "pages": pages, "dtype": dtype, "absent": absent}


def _attention(name, seqs, shortest, longest, heads, kv_heads, head_dim, page, dtype="bf16", window=0, packed=False):
    return {"name": name, "kind": "attention", "seqs": seqs, "shortest": shortest, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "window": window, "packed": packed}


def _linear(name, tokens, k, outputs, high, dtype="bf16", bias=False, activation="none", residual=False):
    return {"name": name, "kind": "linear", "tokens": tokens, "k": k, "outputs": outputs, "high": high, "dtype": dtype,
            "bias": bias, "activation": activation, "residual": residual}


def listed():
    qwen, mistral = dict(heads=28, kv_heads=4, head_dim=128), dict(heads=32, kv_heads=8, head_dim=128)
    return [
        # One user's decode step: the smallest call, where the launch is most of it.
        _norm("norm_decode_1", 1, 3584),
        # An odd batch of a model that norms a block's output and gates it by channel before the residual.
        _norm("norm_gated_77", 77, 2432, "fp16", post=True, gate="channel", scale=0.25),
        # A full prefill chunk: memory decides.
        _norm("norm_prefill_2048", 2048, 3584),
        # Keys and values of a decode batch of 128, three of its rows padding.
        _cache("write_decode_128", "write", 128, 4, 128, 16, 512, absent=3),
        # Keys and values of a prefill chunk.
        _cache("write_prefill_2048", "write", 2048, 8, 128, 16, 256, "fp16"),
        # A cached prefix read back for a prefill chunk behind it; an odd number of tokens, narrow heads.
        _cache("read_prefix_5003", "read", 5003, 8, 64, 32, 256),
        # One user's decode step in the middle of an answer.
        _attention("attention_1", 1, 1000, 1000, page=16, **qwen),
        # A busy server: prompts of very different lengths, one just begun; output for a quantised o_proj.
        _attention("attention_ragged_37", 37, 1, 4099, page=32, dtype="fp16", packed=True, **mistral),
        # A full batch a little behind prompts of 1024 tokens.
        _attention("attention_128", 128, 1024, 1150, page=16, **qwen),
        # Few users with long documents: the axis to split is the cache's.
        _attention("attention_long_4", 4, 32768, 32768, page=16, **qwen),
        # qkv_proj of a decode batch, with its bias.
        _linear("linear_bias_16", 16, 3584, 4608, 512, bias=True),
        # down_proj of a ragged prompt, added to the residual stream.
        _linear("linear_residual_777", 777, 18944, 3584, 384, "fp16", residual=True),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "write", "read", "attention", "attention", "attention", "linear", "linear"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "norm":
        post, gate = rng.random() < 0.3, rng.choice(("none", "none", "none", "channel", "element", "token"))
        case = _norm("", _log_int(rng, 1, 2048), 128 * rng.randint(4, 28), dtype, rng.random() < 0.9, post, gate,
                     rng.choice((1.0, 1.0, 0.25, 1.4)), rng.random() < 0.8)
    elif kind in ("write", "read"):
        page, tokens = rng.choice((16, 32, 64)), _log_int(rng, 1, 4096)
        case = _cache("", kind, tokens, rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128)), page,
                      -(-tokens * 5 // (4 * page)) + rng.randint(1, 64), dtype, rng.choice((0, 0, tokens // 8)))
    elif kind == "attention":
        kv_heads, head_dim, seqs = rng.choice((1, 2, 4, 4, 8)), rng.choice((64, 128, 128)), _log_int(rng, 1, 128)
        longest = _log_int(rng, 1, max(16, min(32768, _MOST_CACHED // (seqs * kv_heads * head_dim))))
        group = rng.choice((1, 2, 4, 4, 5, 7, 8, 12))
        packed = kv_heads * group * head_dim % 128 == 0 and rng.random() < 0.3
        case = _attention("", seqs, rng.choice((longest, longest, max(1, longest // 20), 1)), longest, kv_heads * group,
                          kv_heads, head_dim, rng.choice((16, 16, 32, 64)), dtype,
                          rng.choice((0, 0, 0, max(1, longest // 3))), packed)
    else:
        outputs = _log_int(rng, 640, 12000)
        case = _linear("", _log_int(rng, 1, 777), 128 * _log_int(rng, 4, 48), outputs,
                       round(outputs * rng.choice((0.05, 0.1, 0.1, 0.2))), dtype, rng.random() < 0.6,
                       rng.choice(("none", "none", "relu", "silu", "gelu", "gelu_tanh")), rng.random() < 0.5)
    del case["name"]
    return case


# -- what a program has in hand ---------------------------------------------------------------------------------------------


def _power(e):
    """2^e as fp32, e from -126 to 127."""
    return ((e + 127) << 23).view(torch.float32)


def _exponents(amax, top):
    """The smallest e with amax 2^-e <= top (448 or 6), 0 for a zero."""
    mantissa, e = torch.frexp(amax.float())
    limit, shift = math.frexp(top)
    return torch.where(amax > 0, e - shift + (mantissa > limit), torch.zeros_like(e)).clamp(min=-126).int()


def _mxfp8(v):
    """E4M3 codes [..., k] and exponents [..., k / 32] of fp32 values."""
    groups = v.unflatten(-1, (-1, 32))
    e = _exponents(groups.abs().amax(-1), 448)
    return (groups * _power(-e).unsqueeze(-1)).to(torch.float8_e4m3fn).flatten(-2), e


def _representable(w, fp4):
    """The nearest values that MXFP4 or MXFP8 holds exactly."""
    groups = w.unflatten(-1, (-1, 32))
    scale = _power(_exponents(groups.abs().amax(-1), 6 if fp4 else 448)).unsqueeze(-1)
    v = groups / scale
    if fp4:
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=w.device)
        v = grid[torch.bucketize(v.abs(), (grid[1:] + grid[:-1]) / 2)] * v.sign()
    else:
        v = v.to(torch.float8_e4m3fn).float()
    return (v * scale).flatten(-2)


def _views(data, page, head_dim):
    """Bytes of key codes and value codes [pages, heads, page, head_dim / 32, 8, 4] in the order of their elements, and scales [pages, heads, page, 2, head_dim / 32]."""
    groups, size = head_dim // 32, page * head_dim
    codes = [data[..., i * size:(i + 1) * size].unflatten(-1, (page, 8, groups, 4)).transpose(-2, -3) for i in (0, 1)]
    return codes[0], codes[1], data[..., 2 * size:].unflatten(-1, (page, 2, groups))


def _values(keys, values, scales):
    return {"k": keys.view(torch.float8_e4m3fn), "v": values.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


def _page_bytes(page, head_dim):
    return page * (2 * head_dim + head_dim // 16)


def _keys(shape, generator, dtype):
    """Keys of a trained model have a few channels far larger than the rest."""
    k = torch.randn(shape, device="cuda", generator=generator)
    k[..., :: shape[-1] // 4] *= 4
    return k.to(dtype)


class _State:
    """Inputs, and the layer or the cache; a layer's device memory is given back with it."""
    layer = None

    def __init__(self, case):
        self.case = case

    def __del__(self):
        if self.layer is not None:
            self.layer.close()


def _lengths(case, seed=None):
    """Lengths between the shortest and the longest, evenly by their logarithm; `seed` shuffles them."""
    n, low, high = case["seqs"], case["shortest"], case["longest"]
    lengths = [round(low * (high / low) ** (i / (n - 1))) if n > 1 else high for i in range(n)]
    if seed is not None:
        random.Random(seed).shuffle(lengths)
    return lengths


def _seen(length, window):
    return min(length, window) if window else length


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    state = _State(case)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=generator)

    if kind == "norm":
        rows, k = case["rows"], case["k"]
        x = randn(rows, k)
        x[:, :: k // 16] *= 20
        state.x = x.to(dtype)
        state.weight = (1 + 0.2 * randn(k)).to(dtype)
        state.residual = (3 * randn(rows, k)).to(dtype) if case["residual"] else None
        state.post = (1 + 0.2 * randn(k)).to(dtype) if case["post"] else None
        shape = {"none": None, "channel": (k,), "element": (rows, k), "token": (rows, 1)}[case["gate"]]
        state.gate = torch.tanh(randn(*shape)).to(dtype) if shape else None
    elif kind in ("write", "read"):
        heads, head_dim, page, pages, tokens = case["kv_heads"], case["head_dim"], case["page"], case["pages"], case["tokens"]
        state.data = torch.zeros(pages, heads, _page_bytes(page, head_dim), dtype=torch.uint8, device="cuda")
        slots = torch.randperm(pages * page // 16, device="cuda", generator=generator)   # runs of sixteen, as pages give them
        slots = (slots[: -(-tokens // 16)].unsqueeze(1) * 16 + torch.arange(16, device="cuda")).flatten()[:tokens]
        state.slots = slots.clone()
        if case["absent"]:
            state.slots[torch.randperm(tokens, device="cuda", generator=generator)[: case["absent"]]] = -1
        if kind == "write":   # slices of the output of qkv_proj
            qkv = randn(tokens, 4 * heads * head_dim).to(dtype)
            state.k, state.v = (qkv[:, i * heads * head_dim:(i + 1) * heads * head_dim].unflatten(1, (heads, head_dim)) for i in (2, 3))
            state.k.copy_(_keys((tokens, heads, head_dim), generator, dtype))
        else:
            _fill(state.data, page, head_dim, generator)
    elif kind == "attention":
        heads, head_dim, page, seqs = case["kv_heads"], case["head_dim"], case["page"], case["seqs"]
        lengths = _lengths(case, seed)
        needed = [-(-n // page) for n in lengths]
        state.data = torch.empty(sum(needed) + 8, heads, _page_bytes(page, head_dim), dtype=torch.uint8, device="cuda")
        _fill(state.data, page, head_dim, generator)
        order = torch.randperm(sum(needed) + 8, generator=torch.Generator().manual_seed(seed)).int()
        table, at = torch.zeros(seqs, max(needed), dtype=torch.int32), 0
        for i, n in enumerate(needed):
            table[i, :n] = order[at:at + n]
            at += n
        state.table, state.lengths = table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
        qkv = (2 * randn(seqs, case["heads"] + 2 * heads, head_dim)).to(dtype)
        state.q = qkv[:, : case["heads"]]
    else:
        tokens, k, outputs = case["tokens"], case["k"], case["outputs"]
        x = randn(tokens, k)
        x[:, torch.randperm(k, device="cuda", generator=generator)[: -(-k // 100)]] *= 20
        state.x = x.to(dtype)
        ids = torch.sort(torch.randperm(outputs, device="cuda", generator=generator)[: case["high"]]).values
        w = 0.02 * randn(outputs, k)
        weight = _representable(w, True)
        weight[ids] = _representable(w[ids], False)
        state.weight = weight.to(dtype)
        state.bias = randn(outputs).to(dtype) if case["bias"] else None
        state.residual = (3 * randn(tokens, outputs)).to(dtype) if case["residual"] else None
        if own:   # the layer that a program packs once from these weights
            state.layer = _framework()[1].DualLinear(state.weight, ids)
    if own and kind in ("write", "read", "attention"):
        state.cache = _framework()[0].PagedCache(state.data, case["page"], case["head_dim"])
    return state


def _fill(data, page, head_dim, generator):
    """Keys and values in every entry of a cache."""
    keys, values, scales = _views(data, page, head_dim)
    shape = (data.shape[1], page, head_dim)
    for begin in range(0, data.shape[0], 1024):
        part = slice(begin, min(begin + 1024, data.shape[0]))
        n = part.stop - begin
        made = (_keys((n,) + shape, generator, torch.float32), torch.randn((n,) + shape, device="cuda", generator=generator))
        for i, (to, v) in enumerate(zip((keys, values), made)):
            codes, e = _mxfp8(v)
            to[part] = codes.view(torch.uint8).unflatten(-1, to.shape[3:])
            scales[part, :, :, i] = (e + 127).to(torch.uint8)


# -- the plain forms --------------------------------------------------------------------------------------------------------


def _scale_atoms(e):
    """Scale bytes as the GEMM reads them: atoms of 128 rows x 4 groups, [rows % 32][rows / 32][4] in each; rows behind the last one hold 2^0."""
    rows, groups = e.shape
    full = e.new_zeros(-(-rows // 128) * 128, groups)
    full[:rows] = e
    return (full.view(-1, 4, 32, groups // 4, 4).permute(0, 3, 2, 1, 4) + 127).to(torch.uint8).flatten().view(torch.float8_e8m0fnu)


def _plain_norm(s):
    y, eps = s.x.float(), 1e-6
    if s.post is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * s.post.float()
    if s.gate is not None:
        y = y * s.gate.float()
    y = s.case["scale"] * y
    if s.residual is not None:
        y = y + s.residual.float()
    stream = y.to(s.x.dtype)
    h = stream.float()
    n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * s.weight.float()
    if not s.case["packed"]:
        return {"normed": n.to(s.x.dtype), "stream": stream}
    codes, e = _mxfp8(n)
    return {"codes": codes, "scales": _scale_atoms(e), "stream": stream}


def _plain_write(s):
    page = s.case["page"]
    keys, values, scales = _views(s.data, page, s.case["head_dim"])
    tokens = torch.arange(s.slots.numel(), device="cuda")
    tokens = torch.where(s.slots >= 0, tokens, (s.slots >= 0).int().argmax())   # a padding row writes another row's entry again
    slots = s.slots[tokens]
    at, offset = slots // page, slots % page
    for i, (to, v) in enumerate(((keys, s.k), (values, s.v))):
        codes, e = _mxfp8(v.float())
        to[at, :, offset] = codes.view(torch.uint8).unflatten(-1, to.shape[3:])[tokens]
        scales[at, :, offset, i] = (e + 127).to(torch.uint8)[tokens]
    return _values(keys, values, scales)


def _dequantised(data, page, head_dim, at, offset):
    """Keys and values, fp32 [..., heads, head_dim], of the entries (at, offset)."""
    keys, values, scales = _views(data, page, head_dim)
    scale = _power(scales[at, :, offset].int() - 127)
    return tuple((codes[at, :, offset].view(torch.float8_e4m3fn).float().flatten(-2) * scale[..., i, :].unsqueeze(-1)).flatten(-2) for i, codes in enumerate((keys, values)))


def _plain_read(s):
    page = s.case["page"]
    slots = s.slots.clamp(min=0)
    there = (s.slots >= 0).view(-1, 1, 1)
    k, v = _dequantised(s.data, page, s.case["head_dim"], slots // page, slots % page)
    return {"k": (k * there).to(_DTYPES[s.case["dtype"]]), "v": (v * there).to(_DTYPES[s.case["dtype"]])}


def _plain_attention(s):
    case = s.case
    page, head_dim, kv_heads, seqs = case["page"], case["head_dim"], case["kv_heads"], case["seqs"]
    position = torch.arange(s.table.shape[1] * page, device="cuda")
    k, v = _dequantised(s.data, page, head_dim, s.table.long()[:, position // page], (position % page).expand(seqs, -1))
    q = s.q.float().view(seqs, kv_heads, -1, head_dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * head_dim ** -0.5
    length = s.lengths.view(-1, 1)
    seen = position < length
    if case["window"]:
        seen &= position >= length - case["window"]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (torch.matmul(p, v.transpose(1, 2)) / p.sum(-1, keepdim=True)).reshape(seqs, -1, head_dim)
    if not case["packed"]:
        return {"out": out.to(s.q.dtype)}
    codes, e = _mxfp8(out.flatten(1))
    return {"codes": codes, "scales": _scale_atoms(e)}


def _activated(name, y):
    if name == "relu":
        return y.clamp(min=0)
    if name == "silu":
        return y / (1 + torch.exp(-y))
    if name == "gelu":
        return 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    return y


def _plain_linear(s):
    codes, e = _mxfp8(s.x.float())
    x = (codes.float().unflatten(-1, (-1, 32)) * _power(e).unsqueeze(-1)).flatten(-2)
    y = torch.matmul(x, s.weight.float().t())
    if s.bias is not None:
        y = y + s.bias.float()
    y = _activated(s.case["activation"], y)
    if s.residual is not None:
        y = y + s.residual.float()
    return {"y": y.to(s.x.dtype)}


# -- one pass ---------------------------------------------------------------------------------------------------------------


def _own(s):
    case, kind = s.case, s.case["kind"]
    if kind == "norm":
        producer = _framework()[2]
        call = producer.norm_pack if case["packed"] else producer.norm
        got = call(s.x, s.weight, 1e-6, s.residual, gate=s.gate, scale=case["scale"], post_weight=s.post)
        if not case["packed"]:
            return {"normed": got[0], "stream": got[1]}
        return {"codes": got[0].view(torch.float8_e4m3fn), "scales": got[1].view(torch.float8_e8m0fnu), "stream": got[2]}
    if kind == "linear":
        return {"y": s.layer.linear(s.x, s.bias, case["activation"], s.residual)}
    if kind == "write":
        s.cache.write(s.k, s.v, s.slots)
        return _values(*_views(s.data, case["page"], case["head_dim"]))
    if kind == "read":
        return dict(zip(("k", "v"), s.cache.read(s.slots, _DTYPES[case["dtype"]])))
    if not case["packed"]:
        return {"out": s.cache.attention(s.q, s.table, s.lengths, window=case["window"])}
    codes, scales = s.cache.attention_pack(s.q, s.table, s.lengths, window=case["window"])
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


def run(state):
    if own:
        return _own(state)
    plain = {"norm": _plain_norm, "write": _plain_write, "read": _plain_read, "attention": _plain_attention, "linear": _plain_linear}
    return plain[state.case["kind"]](state)


def work(case):
    kind = case["kind"]
    if kind == "norm":
        cells = case["rows"] * case["k"]
        gates = {"none": 0, "channel": case["k"], "element": cells, "token": case["rows"]}[case["gate"]]
        changed = case["residual"] or case["post"] or gates or case["scale"] != 1.0
        moved = 2 * cells * (1 + case["residual"] + bool(changed)) + 2 * gates + 2 * case["k"] * (1 + case["post"])
        return {"bytes": moved + cells * (33 / 32 if case["packed"] else 2), "flops": 0}
    if kind in ("write", "read"):
        cells = (case["tokens"] - case["absent"]) * case["kv_heads"] * case["head_dim"] * 2
        written = cells if kind == "write" else case["tokens"] * case["kv_heads"] * case["head_dim"] * 2   # 16-bit values on the other side
        return {"bytes": cells * 33 / 32 + 2 * written + 8 * case["tokens"], "flops": 0}
    if kind == "attention":
        seen = sum(_seen(n, case["window"]) for n in _lengths(case))
        cells = case["seqs"] * case["heads"] * case["head_dim"]
        pages = sum(-(-_seen(n, case["window"]) // case["page"]) for n in _lengths(case))
        return {"bytes": seen * case["kv_heads"] * case["head_dim"] * 2 * 33 / 32 + cells * (2 + (33 / 32 if case["packed"] else 2)) + 4 * pages,
                "flops": 4 * seen * case["heads"] * case["head_dim"]}
    m, n, k = case["tokens"], case["outputs"], case["k"]
    weights = (n - case["high"]) * k / 2 + case["high"] * k + n * k / 32 + 4 * n
    return {"bytes": weights + 2 * m * k + 2 * m * n * (1 + case["residual"]) + 2 * n * case["bias"], "flops": 2 * m * n * k}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------------


def _nearest_mxfp8(v):
    """(E4M3 values, powers of two) of the rows of a 64-bit matrix, from the definition of the formats."""
    top = v.reshape(*v.shape[:-1], -1, 32).abs().max(-1, keepdim=True).values
    e = torch.where(top > 0, torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 448)), torch.zeros_like(top))
    e = torch.where(top * 2.0 ** -e > 448, e + 1, e)
    e = torch.where((top > 0) & (top * 2.0 ** (1 - e) <= 448), e - 1, e).clamp(min=-127)
    u = v.reshape(*v.shape[:-1], -1, 32) * 2.0 ** -e
    binade = torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6)))
    step = 2.0 ** (binade - 3)
    return (torch.round(u / step) * step).reshape(v.shape), 2.0 ** e.squeeze(-1)


def _in_atoms(scales):
    rows, groups = scales.shape
    out = torch.ones(-(-rows // 128), groups // 4, 32, 4, 4, dtype=torch.float64, device=scales.device)
    row = torch.arange(rows, device=scales.device)
    out[row // 128, :, row % 32, row % 128 // 32] = scales.reshape(rows, -1, 4)
    return out.flatten()


def _entry_order(data, case):
    """Positions in a page record of the elements d = 0 ... of the keys of its first token."""
    groups = case["head_dim"] // 32
    d = torch.arange(case["head_dim"], device=data.device)
    return (d % 32 // 4) * 4 * groups + d // 32 * 4 + d % 4


def _code_values(codes):
    """E4M3 bytes in 64 bits."""
    b = codes.long()
    exponent, mantissa = b >> 3 & 15, (b & 7).double()
    value = torch.where(exponent > 0, (8 + mantissa) * 2.0 ** (exponent.double() - 10), mantissa * 2.0 ** -9)
    return torch.where(b >= 128, -value, value)


def _entries(data, case, pages, offsets):
    """Keys and values in 64 bits, [entries, heads, head_dim]."""
    page, head_dim = case["page"], case["head_dim"]
    order, groups, got = _entry_order(data, case), head_dim // 32, []
    record = data[pages.long()]                                              # [entries, heads, bytes]
    rows = torch.arange(record.shape[0], device=data.device)[:, None, None]
    heads = torch.arange(record.shape[1], device=data.device)[None, :, None]
    offsets = offsets.long()[:, None, None]
    for i in (0, 1):
        codes = record[rows, heads, i * page * head_dim + offsets * head_dim + order]
        scale = record[rows, heads, 2 * page * head_dim + (offsets * 2 + i) * groups + torch.arange(groups, device=data.device)]
        got.append(_code_values(codes) * (2.0 ** (scale.double() - 127)).repeat_interleave(32, -1))
    return got


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        def rms(t):
            return torch.sqrt((t * t).sum(-1, keepdim=True) / t.shape[-1] + 1e-6)
        h = s.x.double()
        if case["post"]:
            h = h / rms(h) * s.post.double()
        h = h * case["scale"] * (1 if s.gate is None else s.gate.double()) + (0 if s.residual is None else s.residual.double())
        rounded = h.to(s.x.dtype).double()
        n = rounded / rms(rounded) * s.weight.double()
        if not case["packed"]:
            return {"normed": n, "stream": h}
        values, scales = _nearest_mxfp8(n)
        return {"codes": values, "scales": _in_atoms(scales), "stream": h}
    if kind == "write":
        page, groups = case["page"], case["head_dim"] // 32
        shape = (case["pages"], case["kv_heads"], page)
        k, v = (torch.zeros(shape + (groups, 8, 4), dtype=torch.float64, device="cuda") for _ in (0, 1))
        scales = torch.full(shape + (2, groups), 2.0 ** -127, dtype=torch.float64, device="cuda")
        for i, (to, x) in enumerate(((k, s.k), (v, s.v))):
            values, powers = _nearest_mxfp8(x.double())
            for token, slot in enumerate(s.slots.tolist()):
                if slot >= 0:
                    to[slot // page, :, slot % page] = values[token].reshape(-1, groups, 8, 4)
                    scales[slot // page, :, slot % page, i] = powers[token]
        return {"k": k, "v": v, "scales": scales}
    if kind == "read":
        slots = s.slots.clamp(min=0)
        there = (s.slots >= 0).double()[:, None, None]
        k, v = _entries(s.data, case, slots // case["page"], slots % case["page"])
        return {"k": k * there, "v": v * there}
    if kind == "attention":
        group, rows = case["heads"] // case["kv_heads"], []
        for i, length in enumerate(s.lengths.tolist()):
            position = torch.arange(length - _seen(length, case["window"]), length, device="cuda")
            k, v = _entries(s.data, case, s.table[i, position // case["page"]], position % case["page"])
            q = s.q[i].double().reshape(case["kv_heads"], group, case["head_dim"])
            p = torch.softmax(torch.einsum("hgd,thd->hgt", q, k) / math.sqrt(case["head_dim"]), -1)
            rows.append(torch.einsum("hgt,thd->hgd", p, v).reshape(case["heads"], case["head_dim"]))
        out = torch.stack(rows)
        if not case["packed"]:
            return {"out": out}
        values, scales = _nearest_mxfp8(out.flatten(1))
        return {"codes": values, "scales": _in_atoms(scales)}
    values, scales = _nearest_mxfp8(s.x.double())
    y = torch.einsum("mk,nk->mn", values * scales.repeat_interleave(32, -1), s.weight.double())
    if case["bias"]:
        y = y + s.bias.double()
    name = case["activation"]
    if name == "relu":
        y = torch.maximum(y, torch.zeros_like(y))
    elif name == "silu":
        y = y * torch.sigmoid(y)
    elif name in ("gelu", "gelu_tanh"):
        y = torch.nn.functional.gelu(y, approximate="tanh" if name == "gelu_tanh" else "none")
    return {"y": y + (s.residual.double() if case["residual"] else 0)}
