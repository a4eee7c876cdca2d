"""A paged key-value cache in MXFP8 and attention of one new token a sequence over it.

With the linears in MXFP4/MXFP8 the cache is the largest 16-bit operand of a decode step.  Here keys and values are
quantised as they are written, with the rule of `native.pack` (E4M3 codes, one E8M0 scale per 32 elements of a head: 1.03
bytes an element), and read by an attention kernel that multiplies the codes themselves.  Its output can leave as the MXFP8
input of a quantised o_proj, as SwiGLU's does for down_proj (`producer.silu_pack`).

    cache = PagedCache.allocate(pages, page_size=16, kv_heads=4, head_dim=128)
    cache.write(k, v, slots)                                   # slot = page * page_size + place in the page
    y = cache.attention(q, page_table, lengths)                # or
    y = o_proj.run_packed(*cache.attention_pack(q, page_table, lengths))

All calls run on the current stream of the cache's device, allocate only their results and workspace and may be captured in a
CUDA graph.  They are forward only.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native
from .native import DTYPES, _differentiated, _held, _on_device, _stream, check, library, scale_size


class Cache(C.Structure):
    """`hg_cache` of include/hygemm.h."""
    _fields_ = [("data", C.c_void_p), ("pages", C.c_int), ("kv_heads", C.c_int), ("page_size", C.c_int), ("head_dim", C.c_int)]


class AttentionCall(C.Structure):
    """`hg_attention_call` of include/hygemm.h."""
    _fields_ = [("q", C.c_void_p), ("table", C.c_void_p), ("lengths", C.c_void_p), ("out", C.c_void_p), ("codes", C.c_void_p),
                ("scales", C.c_void_p), ("lse", C.c_void_p), ("workspace", C.c_void_p), ("q_stride", C.c_int64),
                ("table_stride", C.c_int64), ("seqs", C.c_int), ("heads", C.c_int), ("table_width", C.c_int),
                ("window", C.c_int), ("scale", C.c_float)]


def page_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one page of one head."""
    return page_size * (2 * head_dim + head_dim // 16)


class PagedCache:
    """`data` is uint8 `[pages, kv_heads, page_bytes(page_size, head_dim)]`; include/hygemm.h describes a page.

    head_dim is 64 or 128, page_size a multiple of 16 up to 1024.
    """

    def __init__(self, data: torch.Tensor, page_size: int, head_dim: int):
        if head_dim not in (64, 128):
            raise ValueError("PagedCache requires head_dim 64 or 128")
        if page_size <= 0 or page_size % 16 or page_size > 1024:
            raise ValueError("PagedCache requires a page_size that is a multiple of 16 up to 1024")
        if not (data.is_cuda and data.dtype == torch.uint8 and data.ndim == 3 and data.is_contiguous() and data.numel()
                and data.shape[2] == page_bytes(page_size, head_dim) and data.data_ptr() % 16 == 0):
            raise ValueError("PagedCache requires contiguous CUDA uint8 [pages, kv_heads, page_bytes(page_size, head_dim)]")
        self.data, self.page_size, self.head_dim = data, page_size, head_dim
        self.pages, self.kv_heads = data.shape[:2]

    @classmethod
    def allocate(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda"):
        """A zeroed cache."""
        if pages <= 0 or kv_heads <= 0 or page_size <= 0 or head_dim <= 0:
            raise ValueError("PagedCache requires pages and heads")
        return cls(torch.zeros((pages, kv_heads, page_bytes(page_size, head_dim)), dtype=torch.uint8, device=device), page_size, head_dim)

    def _struct(self):
        return C.byref(Cache(self.data.data_ptr(), self.pages, self.kv_heads, self.page_size, self.head_dim))

    def _slots(self, slots):
        if not (slots.device == self.data.device and slots.dtype == torch.int64 and slots.ndim == 1 and slots.is_contiguous()):
            raise ValueError("PagedCache requires contiguous int64 slots [tokens] on its device")

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantises `k` and `v` `[tokens, kv_heads, head_dim]` (fp16 or bf16; slices of a qkv output will do) into the entries
        `slots` (int64).  A slot outside the cache, such as the -1 of a padded batch, is left out.  The slots of a call are
        distinct: what an entry named twice holds afterwards is not defined."""
        host = native._host
        if host is not None and host.cache_write(self.data, self.page_size, self.head_dim, k, v, slots):
            return
        shape = (slots.shape[0] if slots.ndim else -1, self.kv_heads, self.head_dim)
        for x in (k, v):
            if not (x.device == self.data.device and x.dtype in DTYPES and x.dtype == k.dtype and x.shape == shape):
                raise ValueError("PagedCache.write requires FP16/BF16 keys and values [tokens, kv_heads, head_dim] on its device")
            if x.numel() and (x.stride(2) != 1 or x.data_ptr() % 8 or x.stride(0) % 4 or x.stride(1) % 4):
                raise ValueError("PagedCache.write requires contiguous heads aligned to 8 bytes")
        self._slots(slots)
        if not _held(self.data, k, v, slots):
            raise ValueError("PagedCache.write requires operands in memory")
        if _differentiated(k, v):
            raise ValueError("PagedCache.write has no gradient")
        if not shape[0]:
            return
        strides = (C.c_int64 * 4)(k.stride(0), k.stride(1), v.stride(0), v.stride(1))
        with _on_device(self.data.device):
            check(library().hg_cache_write(self._struct(), k.data_ptr(), v.data_ptr(), strides, slots.data_ptr(), shape[0],
                                           DTYPES[k.dtype], _stream(self.data.device)))

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        """The entries `slots` as `(k, v)`, each `[tokens, kv_heads, head_dim]` in `dtype`; zeros for a slot outside the cache."""
        if native._host is not None and dtype in DTYPES:
            got = native._host.cache_read(self.data, self.page_size, self.head_dim, slots, DTYPES[dtype])
            if got is not None:
                return got
        self._slots(slots)
        if dtype not in DTYPES:
            raise ValueError("PagedCache.read gives FP16 or BF16")
        if not _held(self.data, slots):
            raise ValueError("PagedCache.read requires operands in memory")
        tokens = slots.shape[0]
        k, v = (torch.empty((tokens, self.kv_heads, self.head_dim), dtype=dtype, device=self.data.device) for _ in (0, 1))
        if tokens:
            with _on_device(self.data.device):
                check(library().hg_cache_read(self._struct(), k.data_ptr(), v.data_ptr(), slots.data_ptr(), tokens, DTYPES[dtype],
                                              _stream(self.data.device)))
        return k, v

    def attention(self, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, scale: float | None = None,
                  window: int = 0, lse: bool = False):
        """Attention of one query a sequence: `q` `[seqs, heads, head_dim]` in fp16 or bf16 (rows may be strided),
        `page_table` int32 `[seqs, pages a sequence has at most]` (rows may be strided), `lengths` int32 `[seqs]`, the new
        token's entry included.  `heads` is a multiple of kv_heads; `scale` defaults to head_dim ** -0.5; a `window` lets a
        sequence see its last `window` positions only.

        Returns `[seqs, heads, head_dim]` in q's dtype, and with `lse` the fp32 logarithms of the sums of weights as well.  A
        sequence that sees nothing (length 0) gives zeros and minus infinity.  A length beyond the table is cut to it, and the
        positions of a page number outside the cache (-1, say, where a page was given up) are left out.  What the table holds
        behind a sequence's last page, and the cache behind its last position, has no influence, NaNs included.
        The weight of a position times the scale of 32 of its channels is rounded to 11 bits; where that is less than 2^-21 of the largest weight
        times the largest scale that these channels have in the sequence, it is off by up to 2^-32 of the latter (`attention_pack` adds what the rounding
        left).  Channels that hold only zeros change nothing of the others, but a head padded with 32 of them takes a quarter longer.
        How the work is spread over the device is chosen by the table's width, so a table far wider than its sequences costs a few us
        (one sequence of 1000 positions 5.3 us with 64 columns, 10.1 with 2048); `page_table[:, :n]` will do.
        """
        return self._attend(q, page_table, lengths, scale, window, lse, False)

    def attention_pack(self, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, scale: float | None = None,
                       window: int = 0, lse: bool = False):
        """The same with the output quantised from its fp32 sums as the `[seqs, heads * head_dim]` input of a hybrid linear: `(q, sf)`
        for `DualLinear.run_packed`."""
        if q.ndim == 3 and (q.shape[1] * q.shape[2]) % 128:
            raise ValueError("PagedCache.attention_pack requires heads * head_dim divisible by 128")
        return self._attend(q, page_table, lengths, scale, window, lse, True)

    def _attend(self, q, page_table, lengths, scale, window, lse, packed):
        if native._host is not None:
            got = native._host.attention(self.data, self.page_size, self.head_dim, q, page_table, lengths, scale, window, lse, packed)
            if got is not None:
                return got
        device = self.data.device
        if not (q.device == device and q.dtype in DTYPES and q.ndim == 3 and q.shape[2] == self.head_dim and q.shape[1]
                and q.shape[1] % self.kv_heads == 0):
            raise ValueError("PagedCache.attention requires FP16/BF16 queries [seqs, heads, head_dim] on its device, heads a multiple of kv_heads")
        seqs, heads, _ = q.shape
        if seqs and (q.stride(2) != 1 or (heads > 1 and q.stride(1) != self.head_dim) or (seqs > 1 and q.stride(0) % 8) or q.data_ptr() % 16):
            raise ValueError("PagedCache.attention requires contiguous query rows aligned to 16 bytes")
        if not _held(self.data, q, page_table, lengths):
            raise ValueError("PagedCache.attention requires operands in memory")
        if _differentiated(q):
            raise ValueError("PagedCache.attention has no gradient")
        if not (page_table.device == device and page_table.dtype == torch.int32 and page_table.ndim == 2 and page_table.shape[0] == seqs
                and (page_table.stride(1) == 1 or page_table.shape[1] <= 1)):
            raise ValueError("PagedCache.attention requires an int32 page table [seqs, pages] on its device")
        if not (lengths.device == device and lengths.dtype == torch.int32 and lengths.shape == (seqs,) and lengths.is_contiguous()):
            raise ValueError("PagedCache.attention requires contiguous int32 lengths [seqs] on its device")
        if window < 0:
            raise ValueError("PagedCache.attention requires a window of at least one position, or 0")
        rows, width = seqs, page_table.shape[1]
        window = 0 if window >= width * self.page_size else window
        out = codes = sf = sums = None
        if packed:
            k = heads * self.head_dim
            codes = torch.empty((rows, k), dtype=torch.uint8, device=device)
            sf = torch.empty(scale_size(rows, k), dtype=torch.uint8, device=device)
        else:
            out = torch.empty((rows, heads, self.head_dim), dtype=q.dtype, device=device)
        if lse:
            sums = torch.empty((rows, heads), dtype=torch.float32, device=device)
        if rows:
            lib, cache = library(), self._struct()
            size = lib.hg_attention_workspace(cache, rows, heads, width, window)
            if size < 0:
                check(-1)
            # A fresh workspace per call: under CUDA-graph capture the graph's pool owns it.
            workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
            call = AttentionCall(q.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), out.data_ptr() if out is not None else None,
                                 codes.data_ptr() if packed else None, sf.data_ptr() if packed else None,
                                 sums.data_ptr() if lse else None, workspace.data_ptr() if size else None, q.stride(0) if rows > 1 else 0,
                                 page_table.stride(0), rows, heads, width, window,
                                 self.head_dim ** -0.5 if scale is None else scale)
            with _on_device(device):
                check(lib.hg_attention(cache, C.byref(call), DTYPES[q.dtype], _stream(device)))
        result = (codes, sf) if packed else (out,)
        return result + (sums,) if lse else result if packed else out
