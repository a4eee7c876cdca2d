"""Fused SwiGLU -> MXFP8 producer feeding down_proj.

Mirror of the reference's `integrations/vllm/hygemm_vllm/producer.py` and
`mistral_producer.py`: `silu_pack` turns the `[M, 2I]` gate||up output of the
hybrid gate_up projection straight into E4M3 codes + E8M0 scales (one kernel
instead of silu_and_mul + memset + pack), and `install()` routes Qwen2 /
Llama / Mistral MLPs through `linear_silu` for up to 128 tokens.
"""
from __future__ import annotations

import ctypes as C
import os

import torch

from . import native
from .native import DTYPES, _differentiated, _held, _on_device, _stream, check, library, scale_size
from .ops import _runtimes, linear_silu  # noqa: F401  (re-exported, reference layout)

MAX_FUSED_TOKENS = 128


def silu_pack(x: torch.Tensor, math: int = 0, debug: bool = False):
    """`[rows, 2K]` gate||up -> (`q [rows,K]` uint8, `sf`) (reference: producer.py:11-24).

    math 0 = expf + IEEE division (bit-exact with SiluAndMul followed by pack),
    1/2 = fast intrinsics.  With `debug=True` also returns the 16-bit product.
    """
    if not (x.is_cuda and x.is_contiguous() and x.dtype in DTYPES and x.ndim == 2):
        raise ValueError("SwiGLU pack requires contiguous CUDA FP16/BF16 [rows, 2K]")
    rows, k = x.shape[0], x.shape[1] // 2
    if x.shape[1] != 2 * k or k % 128:
        raise ValueError("SwiGLU pack requires K divisible by 128")
    q = torch.empty((rows, k), device=x.device, dtype=torch.uint8)
    sf = torch.empty(scale_size(rows, k) if rows else 0, device=x.device, dtype=torch.uint8)
    dbg = torch.empty((rows, k), device=x.device, dtype=x.dtype) if debug else None
    if rows:
        fn = library().hg_silu_pack_bf16 if x.dtype == torch.bfloat16 else library().hg_silu_pack
        status = fn(x.data_ptr(), q.data_ptr(), sf.data_ptr(), dbg.data_ptr() if debug else None,
                    rows, k, _stream(x.device), math)
        if status:
            raise RuntimeError(f"SwiGLU MX producer CUDA status {status}")
    return (q, sf, dbg) if debug else (q, sf)


class NormCall(C.Structure):
    """`hg_norm_call` of include/hygemm.h."""
    _fields_ = [(name, C.c_void_p) for name in ("x", "residual", "gate", "post_weight", "weight", "stream_out", "normed", "codes", "scales")] + [
        ("x_stride", C.c_int64), ("residual_stride", C.c_int64), ("gate_stride", C.c_int64), ("rows", C.c_int), ("k", C.c_int),
        ("gate_per_row", C.c_int), ("eps", C.c_float), ("post_eps", C.c_float), ("scale", C.c_float)]


def _rows_of(name, t, x):
    """Checks a 16-bit matrix like `x` whose rows may be strided."""
    if not (t.device == x.device and t.dtype == x.dtype and t.shape == x.shape and t.stride(1) == 1
            and (t.shape[0] <= 1 or t.stride(0) % 8 == 0) and t.data_ptr() % 16 == 0):
        raise ValueError(f"norm requires {name} [rows,K] of one 16-bit type and device, rows contiguous and aligned to 16 bytes")


# What follows is called through the host extension where that takes a call (`native._host`); here is what it does otherwise, and what is
# wrong with a call that neither takes.
def _norm(x, weight, eps, residual, gate, scale, post_weight, post_eps, packed):
    if not (x.is_cuda and x.dtype in DTYPES and x.ndim == 2 and x.shape[1]):
        raise ValueError("norm requires CUDA FP16/BF16 [rows,K]")
    rows, k = x.shape
    if k % (128 if packed else 8) or k > 32768:
        raise ValueError("norm requires K divisible by 8, quantised by 128, and at most 32768")
    _rows_of("x", x, x)
    if residual is not None:
        _rows_of("residual", residual, x)
    for vector in (weight, post_weight):
        if vector is not None and not (vector.device == x.device and vector.dtype == x.dtype and vector.shape == (k,)
                                       and vector.is_contiguous() and vector.data_ptr() % 16 == 0):
            raise ValueError("norm requires weights [K] of x's type and device, aligned to 16 bytes")
    gate_stride = per_row = 0
    if gate is not None:
        if gate.device != x.device or gate.dtype != x.dtype or tuple(gate.shape) not in ((k,), (rows, k), (rows, 1)):
            raise ValueError("norm requires a gate [K], [rows,K] or [rows,1] of x's type and device")
        if gate.ndim == 2:
            gate_stride = gate.stride(0)
        per_row = int(gate.ndim == 2 and gate.shape[1] == 1 and k != 1)
        if not per_row and (gate.stride(-1) != 1 or (rows > 1 and gate_stride % 8) or gate.data_ptr() % 16):
            raise ValueError("norm requires a gate with contiguous rows aligned to 16 bytes")
    if not _held(x, weight, residual, gate, post_weight):
        raise ValueError("norm requires operands in memory")
    if _differentiated(x, weight, residual, gate, post_weight):
        raise ValueError("norm has no gradient")
    scale = C.c_float(scale).value   # as the kernel takes it: whether the stream changes is decided by the same number there
    changed = residual is not None or gate is not None or post_weight is not None or scale != 1.0
    stream = torch.empty((rows, k), dtype=x.dtype, device=x.device) if changed else x
    normed = codes = sf = None
    if packed:
        codes = torch.empty((rows, k), dtype=torch.uint8, device=x.device)
        sf = torch.empty(scale_size(rows, k), dtype=torch.uint8, device=x.device)
    else:
        normed = torch.empty((rows, k), dtype=x.dtype, device=x.device)
    if rows:
        pointers = (x, residual, gate, post_weight, weight, stream if changed else None, normed, codes, sf)
        call = NormCall(*(None if t is None else t.data_ptr() for t in pointers), x.stride(0),
                        residual.stride(0) if residual is not None else 0, gate_stride, rows, k, per_row, eps,
                        eps if post_eps is None else post_eps, scale)
        if rows == 1:   # the stride of a single row says nothing
            call.x_stride = call.residual_stride = 0
            call.gate_stride = 0
        with _on_device(x.device):
            check(library().hg_norm(C.byref(call), DTYPES[x.dtype], _stream(x.device)))
    return (codes, sf, stream) if packed else (normed, stream)


def norm_pack(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None, *,
              gate: torch.Tensor | None = None, scale: float = 1.0, post_weight: torch.Tensor | None = None,
              post_eps: float | None = None):
    """Residual addition, RMS norm and MXFP8 quantisation in one kernel: `(q, sf, h)`.

    `x` `[rows,K]` is a block's output in fp16 or bf16 (rows may be strided, as `residual`'s may), `h` the new residual stream and
    `(q, sf)` the input of the next hybrid linear (`DualLinear.run_packed`):

        y = x, or with `post_weight`  x / sqrt(mean(x^2) + post_eps) * post_weight
        h = residual + scale * gate * y        rounded to x's type
        n = h / sqrt(mean(h^2) + eps) * weight quantised as `native.pack` does, without a rounding to 16 bits before it

    `gate` is `[K]`, `[rows,K]` or `[rows,1]`; `post_eps` defaults to `eps`.  Without residual, gate, scale and post norm `h` is
    `x` itself.  K is a multiple of 128 up to 32768.  Forward only.
    """
    host = native._host
    got = None if host is None else host.norm(x, weight, eps, residual, gate, scale, post_weight, post_eps, True)
    return _norm(x, weight, eps, residual, gate, scale, post_weight, post_eps, True) if got is None else got


def norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None, *,
         gate: torch.Tensor | None = None, scale: float = 1.0, post_weight: torch.Tensor | None = None,
         post_eps: float | None = None):
    """`norm_pack` for a consumer in 16 bits (an unquantised lm_head, say): `(n, h)`.  K is a multiple of 8 up to 32768."""
    host = native._host
    got = None if host is None else host.norm(x, weight, eps, residual, gate, scale, post_weight, post_eps, False)
    return _norm(x, weight, eps, residual, gate, scale, post_weight, post_eps, False) if got is None else got


def _patch(mlp_class, method_types):
    if getattr(mlp_class, "_hygemm_producer_installed", False):
        return
    original = mlp_class.forward
    math = int(os.environ.get("HYGEMM_SILU_MATH", "0"))

    def forward(self, x):
        method = getattr(self.down_proj, "quant_method", None)
        tokens = x.numel() // x.shape[-1]
        if not isinstance(method, method_types) or tokens > MAX_FUSED_TOKENS or getattr(method, "runtime", None) is None:
            return original(self, x)
        if self.down_proj.bias is not None:
            raise ValueError("Fused SwiGLU path does not support a down_proj bias")
        gate_up, _ = self.gate_up_proj(x)
        y = linear_silu(gate_up.reshape(-1, 2 * method.k), method.handle, method.outputs, math)
        y = method.reduce(y)
        return y.reshape(*x.shape[:-1], method.outputs)

    mlp_class.forward = forward
    mlp_class._hygemm_producer_installed = True


def install(llama: bool = False):
    """Patch the MLP forward of Qwen2 (and Llama/Mistral when asked) (reference: producer.py:43-58,
    mistral_producer.py:5-27).  The reference limits the patch to its offline method; here every
    hybrid linear method qualifies."""
    from .quantization import MixedLinearMethod
    from vllm.model_executor.models.qwen2 import Qwen2MLP
    _patch(Qwen2MLP, MixedLinearMethod)
    if llama:
        from vllm.model_executor.models.llama import LlamaMLP
        _patch(LlamaMLP, MixedLinearMethod)
        try:
            from vllm.model_executor.models.mistral import MistralMLP
            _patch(MistralMLP, MixedLinearMethod)
        except ImportError:
            pass
