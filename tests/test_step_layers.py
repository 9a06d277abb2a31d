"""A generate step writes a slot in every layer of its cache: a cache whose keys and values have
too few layers on one side is refused before anything is launched."""

from __future__ import annotations

import pytest
import torch

import bdh_hip_ext as ext
import kernels
from kernels import Mx4

BF = torch.bfloat16


def _step(fn, kr, v_layers):
    B, nh, N, D, cap = 2, 2, 64, 64, 5
    cos, sin = kernels.rope_cos_sin(1, 3, kernels.get_freqs(N))
    w = [torch.zeros(s, dtype=BF) for s in ((nh, N, D), (nh, N, D), (nh * N, D))]
    return fn(torch.zeros(B, D), *w, cos, sin, kr, torch.zeros(v_layers, B, 1, cap, D, dtype=BF), 3)


def _keys(layers, four):
    return Mx4.empty(layers, 2, 2, 5, 64) if four else torch.zeros(layers, 2, 2, 5, 64, dtype=BF)


@pytest.mark.parametrize("n", [1, 3])
def test_too_few_layers(n):
    # (the 4-bit step takes its count from v, the other from kr)
    for fn, kr, v_layers in ((ext.decode_step_mx4, _keys(n, True), n + 1), (ext.decode_step_mx4, _keys(n, False), n + 1),
                             (ext.decode_step_mx4, _keys(n, True), 0), (ext.decode_step, _keys(n + 1, False), n),
                             (ext.decode_step_mx4, _keys(n, True)[0], 1)):
        with pytest.raises(ValueError, match="layers"):
            _step(fn, kr, v_layers)


@pytest.mark.skipif(torch.cuda.is_available(), reason="host tensors are refused the same with a GPU")
def test_enough_layers_pass_that_check():
    for fn, four, n, m in ((ext.decode_step_mx4, True, 2, 2), (ext.decode_step_mx4, True, 3, 2), (ext.decode_step, False, 2, 2),
                           (ext.decode_step, False, 2, 3)):
        with pytest.raises(RuntimeError, match="GPU"):
            _step(fn, _keys(n, four), m)
