"""The eager forms of the 4-bit rows on GPU tensors: scales are powers of two and have to be exact
there too (a device's pow need not give them), so codes and values are the definition's."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mx4_oracle as M

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a ROCm GPU", allow_module_level=True)

import kernels  # noqa: E402
from kernels import Mx4  # noqa: E402

F32, BF = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF])
def test_values_of_every_code_and_scale(dtype):
    s = torch.arange(256, dtype=torch.uint8).view(256, 1)
    c = (torch.arange(16) + 16 * torch.arange(15, -1, -1)).to(torch.uint8).repeat(256, 1)
    want = M.values(Mx4(c, s, 32))
    got = kernels.mx4_dequantize(Mx4(c.cuda(), s.cuda(), 32), dtype, impl="eager").double().cpu().numpy()
    fits = np.abs(want) < 2.0 ** 128
    np.testing.assert_array_equal(got[fits], want[fits])
    assert np.isnan(got[255]).all() and np.isinf(got[~fits & ~np.isnan(want)]).all()


@pytest.mark.parametrize("n", [1, 33, 100])
def test_codes_over_every_scale(n):
    """The rows that are hard to round, at every size a block can have."""
    hard = M.hard_rows(n)
    x = torch.cat([torch.ldexp(hard, torch.tensor(e)) for e in range(-60, 61, 3)] + [hard])
    codes, scales = M.quantize(x.double().numpy())
    m = kernels.mx4_quantize(x.cuda(), impl="eager")
    np.testing.assert_array_equal(m.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(m.codes.cpu().numpy(), M.pack(codes))


def test_products_and_decode_at_every_scale():
    """One nonzero code a row, so that a result is one value: equal to it, whatever the scale."""
    b = torch.arange(1, 254, dtype=torch.uint8)
    codes = torch.zeros(253, 16, dtype=torch.uint8)
    codes[:, 0] = 2  # 1.0
    w = Mx4(codes.cuda(), b.view(-1, 1).cuda(), 32)
    want = 2.0 ** (b.double() - 127)
    a = torch.zeros(1, 32, dtype=BF, device="cuda")
    a[0, 0] = 1
    assert torch.equal(kernels.mx4_gemm(a, w, out_dtype=F32, impl="eager")[0].double().cpu(), want)
    k = Mx4(w.codes.view(1, 1, 253, 16), w.scales.view(1, 1, 253, 1), 32)
    v = torch.eye(253, device="cuda").view(1, 1, 253, 253)
    got = kernels.bdh_attn_decode(a.float().view(1, 1, 1, 32), k, v, impl="eager")
    assert torch.equal(got.flatten().double().cpu(), want)
