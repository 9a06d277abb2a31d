"""Operators on microscaled 4-bit rows: quantisation, RoPE into a 4-bit cache, products with 4-bit weights.

The format is :mod:`kernels.mx4`'s; a decode over 4-bit keys is
``bdh_attn_decode`` with an ``Mx4`` past.  On the GPU each first tries the compiled
binding, which takes arguments that need no preparation; the checks after it say
what is wrong with others, or prepare them.  The backends are those of the
attention (``BDH_ATTN_IMPL``): ``hip`` runs the gfx950 kernels, ``eager`` torch
operations, on any device.  Both give the same codes; products differ in
summation order.  Nothing here has a derivative: inputs and outputs that need gradients
(unless under ``torch.no_grad()``) or carry forward-mode tangents raise ``ValueError``.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import hip_attn
from .attention_dispatch import resolve_attn_impl
from .hip_attn import _last_dim_unit
from .mx4 import (
    _FLOATS,
    Mx4,
    _eager_gemm,
    _eager_quantize,
    _eager_rope,
    _eager_values,
    _float_rows,
    _no_grad,
    _same,
    _unit_out,
)


def mx4_quantize(x: torch.Tensor, out: Optional[Mx4] = None, *, impl: Optional[str] = None) -> Mx4:
    """``x`` (1- to 4-D, float32 or bfloat16) in mx4, blocks along its last dim; ``out`` may be
    rows of a cache (any outer strides)."""
    name = resolve_attn_impl(impl)
    if name == "hip" and x.is_cuda:
        m = Mx4.empty(*x.shape, device=x.device) if out is None and x.dim() > 0 else out
        if hip_attn._require().mx4_quantize_fast(x, m) is not None:
            return m
    _float_rows("mx4_quantize", x)
    _no_grad("mx4_quantize", x)
    if out is None:
        out = Mx4.empty(*x.shape, device=x.device)
    else:
        _same("mx4_quantize out", out, x)
    if name == "eager":
        c, s = _eager_quantize(x)
        out.codes.copy_(c)
        out.scales.copy_(s)
    else:
        hip_attn._require().mx4_quantize(_last_dim_unit(x), out)
    return out


def mx4_dequantize(m: Mx4, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None, *,
                   impl: Optional[str] = None) -> torch.Tensor:
    """The values that ``m`` stands for, in ``dtype`` (float32 or bfloat16: both hold them), or into
    ``out`` (any outer strides)."""
    name = resolve_attn_impl(impl)
    given = out
    if out is None:
        out = torch.empty(m.shape, dtype=dtype, device=m.codes.device)
    if name == "hip" and out.is_cuda and hip_attn._require().mx4_dequantize_fast(m, out) is not None:
        return out
    if given is not None:
        _same("mx4_dequantize", m, out)
    _float_rows("mx4_dequantize", out)
    _no_grad("mx4_dequantize", out)
    if name == "eager":
        return out.copy_(_eager_values(m))
    _unit_out("mx4_dequantize", out)
    return hip_attn._require().mx4_dequantize(m, out)


def mx4_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, slot: Mx4, out: Optional[torch.Tensor] = None, *,
             impl: Optional[str] = None) -> Mx4:
    """RoPE of ``x`` (..., N) into the 4-bit rows ``slot`` (the KV cache's), and, with ``out``, the
    rotated rows rounded to its dtype (the decode's queries).

    The rotation is the adjacent-pair one of ``bdh_rope_rotate`` with fp32 products and sum whatever
    x's dtype; ``slot`` is quantised from the fp32 values.  ``cos`` / ``sin``: float32, broadcastable
    to x, the last dim N."""
    name = resolve_attn_impl(impl)
    if name == "hip" and x.is_cuda and hip_attn._require().mx4_rope_fast(x, cos, sin, slot, out) is not None:
        return slot
    _float_rows("mx4_rope", x)
    _no_grad("mx4_rope", x, cos, sin, out)
    n = x.size(-1)
    if n % 2 != 0:
        raise ValueError(f"RoPE last dim must be even, got {n}")
    if cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError(f"mx4_rope: float32 cos and sin of one shape, got {cos.dtype} {tuple(cos.shape)} and "
                         f"{sin.dtype} {tuple(sin.shape)}")
    if cos.dim() == 0 or cos.size(-1) != n:
        raise ValueError(f"cos/sin last dim of {tuple(cos.shape)} != x last dim {n}")
    _same("mx4_rope slot", slot, x)
    if out is not None:
        _float_rows("mx4_rope out", out)
        if out.shape != x.shape or out.get_device() != x.get_device():
            raise ValueError(f"rope out= must match x shape/device, got {tuple(out.shape)}/{out.device}")
        _unit_out("mx4_rope", out)
    if name == "eager":
        try:
            r = _eager_rope(x, cos.expand(x.shape), sin.expand(x.shape))
        except RuntimeError as exc:
            raise ValueError(f"cos/sin {tuple(cos.shape)} do not broadcast to x {tuple(x.shape)}") from exc
        mx4_quantize(r, slot, impl="eager")
        if out is not None:
            out.copy_(r)
    else:
        hip_attn._require().mx4_rope(_last_dim_unit(x), _last_dim_unit(cos), _last_dim_unit(sin), slot, out)
    return slot


def mx4_gemm(a, wt: Mx4, *, relu: bool = False, mul: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16,
             impl: Optional[str] = None) -> torch.Tensor:
    """``[mul *] [relu](a @ wt^T)`` with 4-bit weights, rounded once to ``out_dtype``.

    ``wt`` (N, K) or, per head, (H, N, K); ``a`` (M, K) or (H, M, K) alike: bfloat16 rows (a head
    stride of 0 shares them), whose products with the weights' values are exact, or an ``Mx4``.
    ``mul`` and ``out``: (M, N) or (H, M, N), float32 or bfloat16, any outer strides."""
    name = resolve_attn_impl(impl)
    if name == "hip" and a.is_cuda and out_dtype in _FLOATS:
        r = hip_attn._require().mx4_gemm_fast(a, wt, relu, mul, out, out_dtype is torch.bfloat16)
        if r is not None:
            return r
    four = isinstance(a, Mx4)
    if not isinstance(wt, Mx4) or wt.codes.dim() not in (2, 3):
        raise ValueError("mx4_gemm: wt an Mx4 (N, K) or (H, N, K)")
    if not four and a.dtype != torch.bfloat16:
        raise ValueError(f"mx4_gemm: a in bfloat16 or an Mx4, got {a.dtype}")
    ashape, wshape = a.shape, wt.shape
    if len(ashape) != len(wshape) or ashape[:-2] != wshape[:-2] or ashape[-1] != wshape[-1]:
        raise ValueError(f"mx4_gemm: a {tuple(ashape)} and wt {wshape} do not match")
    shape, dev = (*ashape[:-1], wshape[-2]), wt.codes.get_device()
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=wt.codes.device)
    elif out.shape != shape:
        raise ValueError(f"mx4_gemm: out {shape} wanted, got {tuple(out.shape)}")
    if mul is not None and mul.shape != shape:
        raise ValueError(f"mx4_gemm: mul {shape} wanted, got {tuple(mul.shape)}")
    if out.dtype not in _FLOATS or (mul is not None and mul.dtype not in _FLOATS):
        raise ValueError("mx4_gemm: mul and out in float32 or bfloat16")
    if ((a.codes if four else a).get_device() != dev or out.get_device() != dev
            or (mul is not None and mul.get_device() != dev)):
        raise ValueError("mx4_gemm: operands on different devices")
    _no_grad("mx4_gemm", None if four else a, mul, out)
    if name == "eager":
        return out.copy_(_eager_gemm(a, wt, relu, mul))
    _unit_out("mx4_gemm", out)
    return hip_attn._require().mx4_gemm(None if four else _last_dim_unit(a), a if four else None, wt,
                                        None if mul is None else _last_dim_unit(mul), relu, out)


__all__ = ["mx4_quantize", "mx4_dequantize", "mx4_rope", "mx4_gemm"]
