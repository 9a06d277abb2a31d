"""The generate step over 4-bit rows has no derivative either: operands that need gradients or carry
forward-mode tangents are refused, as by the operators."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

import bdh_hip_ext as ext
import kernels
from kernels import Mx4

BF = torch.bfloat16
NAMES = ["x", "enc_t", "encv_t", "dec", "cos", "sin", "v"]


def operands():
    B, nh, N, D, cap = 2, 2, 64, 64, 5
    cos, sin = kernels.rope_cos_sin(1, 3, kernels.get_freqs(N))
    return dict(x=torch.zeros(B, D), enc_t=torch.zeros(nh, N, D, dtype=BF), encv_t=torch.zeros(nh, N, D, dtype=BF),
                dec=torch.zeros(nh * N, D, dtype=BF), cos=cos, sin=sin, kr=Mx4.empty(1, B, nh, cap, N),
                v=torch.zeros(1, B, 1, cap, D, dtype=BF), seq_len=3)


@pytest.mark.parametrize("name", NAMES)
def test_operands_with_derivatives(name):
    ops = operands()
    need = dict(ops, **{name: ops[name].clone().requires_grad_()})
    with pytest.raises(ValueError, match="derivative"):
        ext.decode_step_mx4(**need)
    with fwd.dual_level():
        dual = dict(ops, **{name: fwd.make_dual(ops[name].clone(), torch.ones_like(ops[name]))})
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="derivative"):
                ext.decode_step_mx4(**dual)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # (host tensors are refused next)
        ext.decode_step_mx4(**need)
