"""Microscaled 4-bit rows (``Mx4``), their ``eager`` forms, and the decode over a 4-bit past.

A row's elements go in blocks of 32 consecutive ones (the last may be shorter).
An element is a 4-bit E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign),
element 2i in the low half of byte i; a block has one E8M0 scale byte ``b``,
which stands for ``2^(b - 127)``::

    scale    the smallest power of two (from 2^-127 on) that takes the block's
             largest magnitude below 7, so that it rounds to 6 at most
    element  x / scale to the nearest code, ties to the even one

A block that holds an infinity or a NaN has the scale byte 255 and stands for
NaN.  17 bytes hold 32 elements, 17/64 of their bf16.  Rotated ReLU latents lose
0.115 of their norm (0.118, and 2.3 % of their size instead of 1 %, under the
rule that takes the scale from the largest magnitude's exponent alone, where
what rounds above 6 is cut to it).

This module holds the rows and their torch forms; :mod:`kernels.mx4_dispatch` is
the operators' surface.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.forward_ad import unpack_dual

from . import hip_attn

BLOCK = 32
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _blocks(width: int) -> int:
    return -(-width // BLOCK)


class Mx4:
    """Rows in microscaled 4-bit floating point: ``codes`` (..., 16 * blocks) and
    ``scales`` (..., blocks), both uint8 with unit stride in the last dim, for rows of
    ``width`` elements; codes behind a row's end are zero.  Views (``narrow``,
    indexing of outer dims) share memory with their ``Mx4``."""

    __slots__ = ("codes", "scales", "width")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, width: int):
        kb = (width + 31) // 32
        cs, ss = codes.shape, scales.shape
        if width < 0 or len(cs) == 0 or len(ss) == 0 or cs[:-1] != ss[:-1] or cs[-1] != 16 * kb or ss[-1] != kb:
            raise ValueError(f"Mx4: rows of {width} take {16 * kb} code and {kb} scale bytes, got "
                             f"{tuple(cs)} and {tuple(ss)}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"Mx4: codes and scales are uint8, got {codes.dtype} and {scales.dtype}")
        if codes.get_device() != scales.get_device():
            raise ValueError(f"Mx4: codes on {codes.device}, scales on {scales.device}")
        if (codes.stride(-1) != 1 and kb > 0) or (scales.stride(-1) != 1 and kb > 1):
            raise ValueError("Mx4: codes and scales have unit stride in their last dim")
        self.codes, self.scales, self.width = codes, scales, width

    @classmethod
    def empty(cls, *shape: int, device=None) -> "Mx4":
        """Rows of ``shape[-1]`` elements, their memory not set."""
        kb = _blocks(shape[-1])
        return cls._of(torch.empty(*shape[:-1], 16 * kb, dtype=torch.uint8, device=device),
                       torch.empty(*shape[:-1], kb, dtype=torch.uint8, device=device), shape[-1])

    @classmethod
    def _of(cls, codes: torch.Tensor, scales: torch.Tensor, width: int) -> "Mx4":
        """From memory that holds rows already (views of an ``Mx4``)."""
        m = object.__new__(cls)
        m.codes, m.scales, m.width = codes, scales, width
        return m

    @property
    def shape(self) -> tuple:
        return (*self.codes.shape[:-1], self.width)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def dim(self) -> int:
        return self.codes.dim()

    def size(self, dim: Optional[int] = None):
        return self.shape if dim is None else self.shape[dim]

    def _outer(self, dim: int) -> int:
        n = self.codes.dim()
        d = dim + n if dim < 0 else dim
        if not 0 <= d < n - 1:
            raise ValueError(f"Mx4: dim {dim} of {n}-D rows cannot be cut (blocks run along the last one)")
        return d

    def narrow(self, dim: int, start: int, length: int) -> "Mx4":
        d = self._outer(dim)
        return Mx4._of(self.codes.narrow(d, start, length), self.scales.narrow(d, start, length), self.width)

    def __getitem__(self, i: int) -> "Mx4":
        self._outer(0)
        return Mx4._of(self.codes[int(i)], self.scales[int(i)], self.width)

    def __repr__(self) -> str:
        return f"Mx4(shape={self.shape}, device='{self.device}')"


# ------------------------------------------------------------------- eager
def _pow2(b: torch.Tensor) -> torch.Tensor:
    """What scale bytes stand for, 2^(b - 127) or NaN, by their bits: on a GPU torch.ldexp goes by a
    pow that misses powers of two by a step, and codes at a border with it."""
    b = b.int()
    return torch.where(b == 0, 0x00400000, torch.where(b == 255, 0x7FC00000, b << 23)).view(torch.float32)


def _eager_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    n = x.size(-1)
    y = torch.nn.functional.pad(x.float(), (0, -n % BLOCK)).unflatten(-1, (_blocks(n), BLOCK))
    top = y.abs().amax(-1)
    bad = ~torch.isfinite(y).all(-1)
    m, e = torch.frexp(torch.where(bad, 0.0, top))  # m 2^e, 0.5 <= m < 1
    e = torch.where(m > 0, e - 3 + (m >= 0.875).int(), -127).clamp(-127, 127)
    y = y * _pow2(127 - e).unsqueeze(-1)
    a = y.abs()
    i = torch.where(a < 2, torch.round(2 * a), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4))
    i = i.clamp_max(7) + 8 * torch.signbit(y)
    i = torch.where(bad.unsqueeze(-1), 0.0, i).to(torch.uint8).flatten(-2)
    return i[..., 0::2] + 16 * i[..., 1::2], torch.where(bad, 255, e + 127).to(torch.uint8)


def _eager_values(m: Mx4) -> torch.Tensor:
    lut = torch.tensor(_GRID + tuple(-v for v in _GRID), device=m.device)
    v = lut[torch.stack((m.codes & 15, m.codes >> 4), -1).flatten(-2).long()].unflatten(-1, (_blocks(m.width), BLOCK))
    return (v * _pow2(m.scales).unsqueeze(-1)).flatten(-2)[..., : m.width]


def _eager_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    x = x.float()
    x0, x1 = x[..., 0::2], x[..., 1::2]
    y0 = x0 * cos[..., 0::2] - x1 * sin[..., 0::2]
    y1 = x1 * cos[..., 1::2] + x0 * sin[..., 1::2]
    return torch.stack((y0, y1), -1).flatten(-2)


def _eager_gemm(a, wt: Mx4, relu: bool, mul: Optional[torch.Tensor]) -> torch.Tensor:
    a = _eager_values(a) if isinstance(a, Mx4) else a.float()
    y = torch.matmul(a, _eager_values(wt).transpose(-1, -2).contiguous())
    y = torch.relu(y) if relu else y
    return y if mul is None else y * mul.float()


# ------------------------------------------------------------------ checks
_FLOATS = (torch.float32, torch.bfloat16)


def _float_rows(name: str, t: torch.Tensor) -> None:
    if t.dtype not in _FLOATS:
        raise ValueError(f"{name}: float32 or bfloat16 rows, got {t.dtype}")
    if not 1 <= t.dim() <= 4:
        raise ValueError(f"{name}: rows of 1 to 4 dims, got shape {tuple(t.shape)}")


def _no_grad(name: str, *ts: Optional[torch.Tensor]) -> None:
    """Operands, outputs among them, that need gradients or carry a forward-mode tangent."""
    grad = torch.is_grad_enabled()
    for t in ts:
        if t is None:
            continue
        if grad and t.requires_grad:
            raise ValueError(f"{name} has no backward: call it under torch.no_grad() or detach its operands")
        if unpack_dual(t).tangent is not None:  # (no_grad does not put these off)
            raise ValueError(f"{name} has no forward-mode derivative: call it on the primal tensors")


def _same(name: str, m: Mx4, t: torch.Tensor) -> None:
    if m.shape != t.shape or m.codes.get_device() != t.get_device():
        raise ValueError(f"{name}: Mx4 of shape {tuple(t.shape)} on {t.device} wanted, got {m}")


def _unit_out(name: str, out: torch.Tensor) -> None:
    if out.stride(-1) != 1 and out.size(-1) > 1:
        raise ValueError(f"{name}: out must have unit stride in its last dim")


def mx4_decode(Q: torch.Tensor, K_past: Mx4, V_past: torch.Tensor, impl: str) -> torch.Tensor:
    """``bdh_attn_decode`` over a 4-bit past (its shape contract; any width)."""
    if impl == "hip" and Q.is_cuda:
        out = hip_attn._require().mx4_decode_fast(Q, K_past, V_past)
        if out is not None:
            return out
    qs, ks, vs = Q.shape, K_past.codes.shape, V_past.shape
    if not (len(qs) == len(ks) == len(vs) == 4 and ks[:2] == qs[:2] and qs[3] == K_past.width
            and vs[0] == qs[0] and vs[2] == ks[2] and (vs[1] == 1 or vs[1] == qs[1])):
        hip_attn._check_decode_shapes(Q, K_past, V_past)  # names what is wrong
    _no_grad("bdh_attn_decode over an Mx4 past", Q, V_past)
    if impl == "eager":
        s = torch.matmul(Q.float(), _eager_values(K_past).transpose(-1, -2).contiguous())
        return torch.matmul(s, V_past.float().expand(-1, Q.size(1), -1, -1)).to(Q.dtype)
    return hip_attn._require().mx4_decode(hip_attn._last_dim_unit(Q), K_past, hip_attn._last_dim_unit(V_past))


__all__ = ["Mx4", "mx4_decode"]
