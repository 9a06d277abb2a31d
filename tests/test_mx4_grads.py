"""The 4-bit operators refuse what autograd would need them for: inputs and outputs that need
gradients, and forward-mode tangents, which they would lose."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

import kernels
import mx4_oracle as M

BF = torch.bfloat16


def operands(device="cpu"):
    x = M.rows((1, 2, 3, 64), 1).to(device)
    cos, sin = (t.to(device) for t in kernels.rope_cos_sin(3, 0, kernels.get_freqs(64)))
    m = kernels.mx4_quantize(x, impl="eager")
    a, mul = M.rows((2, 5, 64), 2, BF).to(device), M.rows((2, 5, 3), 3).to(device)
    return x, cos, sin, m, m[0], a, mul


def calls(device, impl):
    """{name: (call with one operand replaced, that operand)}"""
    x, cos, sin, m, wt, a, mul = operands(device)
    h = dict(impl=impl)
    y = torch.empty_like(mul)
    return {
        "quantize x": (lambda t: kernels.mx4_quantize(t, **h), x),
        "dequantize out": (lambda t: kernels.mx4_dequantize(m, out=t, **h), x.clone()),
        "rope x": (lambda t: kernels.mx4_rope(t, cos, sin, m, **h), x),
        "rope cos": (lambda t: kernels.mx4_rope(x, t, sin, m, **h), cos),
        "rope sin": (lambda t: kernels.mx4_rope(x, cos, t, m, **h), sin),
        "rope out": (lambda t: kernels.mx4_rope(x, cos, sin, m, out=t, **h), torch.empty_like(x)),
        "decode q": (lambda t: kernels.bdh_attn_decode(t, m, x, **h), x[:, :, :1].clone()),
        "decode v": (lambda t: kernels.bdh_attn_decode(x[:, :, :1], m, t, **h), x.clone()),
        "gemm a": (lambda t: kernels.mx4_gemm(t, wt, **h), a),
        "gemm mul": (lambda t: kernels.mx4_gemm(a, wt, mul=t, **h), mul),
        "gemm out": (lambda t: kernels.mx4_gemm(a, wt, out=t, **h), y),
    }


NAMES = list(calls("cpu", "eager"))


@pytest.mark.parametrize("name", NAMES)
def test_operands_that_need_gradients(name):
    call, t = calls("cpu", "eager")[name]
    t = t.clone().requires_grad_()
    was = t.detach().clone()
    with pytest.raises(ValueError):
        call(t)
    assert torch.equal(t.detach().view(torch.uint8), was.view(torch.uint8))
    with torch.no_grad():
        call(t)


@pytest.mark.parametrize("name", NAMES)
def test_operands_with_tangents(name):
    call, t = calls("cpu", "eager")[name]
    with fwd.dual_level():
        dual = fwd.make_dual(t.clone(), torch.ones_like(t))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError):
                call(dual)
        call(t)
    call(t)
