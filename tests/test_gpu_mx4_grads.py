"""The 4-bit operators on the GPU refuse operands that need gradients or carry tangents, by the
compiled binding and by the checks behind it, before a launch."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a ROCm GPU", allow_module_level=True)

import bdh_hip_ext as ext  # noqa: E402
from test_mx4_grads import NAMES, calls  # noqa: E402


@pytest.mark.parametrize("name", NAMES)
def test_operands_that_need_gradients_or_carry_tangents(name):
    call, t = calls("cuda", "hip")[name]
    need = t.clone().requires_grad_()
    was = need.detach().clone()
    before = ext.launch_count()
    with pytest.raises(ValueError):
        call(need)
    with fwd.dual_level():
        dual = fwd.make_dual(t.clone(), torch.ones_like(t))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError):
                call(dual)
    assert ext.launch_count() == before
    assert torch.equal(need.detach().view(torch.uint8), was.view(torch.uint8))
    with torch.no_grad():
        call(need)
    assert ext.launch_count() == before + 1
