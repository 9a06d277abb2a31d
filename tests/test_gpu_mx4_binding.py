"""The 4-bit operators without the compiled binding: the ctypes route gives the same bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a ROCm GPU", allow_module_level=True)

import bdh_hip_ext as ext  # noqa: E402
import kernels  # noqa: E402
import mx4_oracle as M  # noqa: E402
from kernels import Mx4  # noqa: E402

BF, F32 = torch.bfloat16, torch.float32


def _all():
    x = M.rows((2, 3, 40, 96), 1, BF).cuda()
    cos, sin = (t.cuda() for t in kernels.rope_cos_sin(40, 5, kernels.get_freqs(96)))
    m = kernels.mx4_quantize(x, impl="hip")
    into = kernels.mx4_quantize(x, Mx4.empty(2, 3, 50, 96, device="cuda").narrow(2, 4, 40), impl="hip")
    slot, r = Mx4.empty(2, 3, 40, 96, device="cuda"), torch.empty_like(x)
    kernels.mx4_rope(x, cos, sin, slot, out=r, impl="hip")
    q, v = x[:, :, :1].float(), M.rows((2, 1, 40, 32), 2).cuda()
    a, mul = M.rows((3, 70, 96), 3, BF).cuda(), M.rows((70, 3, 40), 4).cuda().permute(1, 0, 2)
    wt = m[0]
    return [m.codes, m.scales, into.codes, into.scales, slot.codes, slot.scales, r,
            kernels.mx4_dequantize(slot, F32, impl="hip"), kernels.mx4_dequantize(m[0][0], impl="hip"),
            kernels.bdh_attn_decode(q, m, v, impl="hip"), kernels.bdh_attn_decode(q.to(BF), m, v, impl="hip"),
            kernels.mx4_gemm(a, wt, relu=True, mul=mul, out_dtype=F32, impl="hip"),
            kernels.mx4_gemm(kernels.mx4_quantize(a[0], impl="hip"), wt[0], impl="hip")]


def test_the_ctypes_route_gives_the_same(monkeypatch):
    assert ext._bind is not None
    before = ext.launch_count()
    want = _all()
    n = ext.launch_count() - before
    monkeypatch.setattr(ext, "_bind", None)
    got = _all()
    assert ext.launch_count() - before == 2 * n
    assert all(torch.equal(a, b) for a, b in zip(got, want))
