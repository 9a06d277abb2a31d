"""Decode and products of the 4-bit operators at lengths where a bound on roundings says little: whole
numbers whose sums fp32 holds exactly, so the results have to be equal (mx4_exact.py says why; that
the comparison sees one missing key or block, test_mx4_exact.py).

A matrix instruction may align its products to the largest of them; here all are multiples of 1/4
below 2^22 / 4, within the 24 bits that an fp32 sum keeps."""

from __future__ import annotations

import pytest
import torch

import mx4_exact as X

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a ROCm GPU", allow_module_level=True)

import bdh_hip_ext as ext  # noqa: E402
import kernels  # noqa: E402
from kernels import Mx4  # noqa: E402

F32, BF = torch.float32, torch.bfloat16


def dev(t):
    return Mx4(t.codes.cuda(), t.scales.cuda(), t.width) if isinstance(t, Mx4) else t.cuda()


@pytest.mark.parametrize("shape", X.DECODE)
def test_decode(shape):
    for qdt in (F32, BF):
        q, k, v = X.decode_operands(*shape, qdt, BF)
        want, k4 = X.decode_want(q, k, v), dev(k)
        for vdt in (BF, F32):
            print("decode", shape, qdt, vdt, flush=True)
            got = kernels.bdh_attn_decode(q.cuda(), k4, v.to(vdt).cuda(), impl="hip")
            assert X.equal(got, want)


def test_decode_in_a_cache():
    """Rows of a cache with room, heads permuted, V rows padded, q off 16 bytes."""
    B, H, S, cap, N, D = 16, 4, 70, 90, 8192, 80
    for qdt in (F32, BF):
        q, k, v = X.decode_operands(B, H, 1, cap, N, D, 1, qdt, BF)
        full = dev(k)
        cache = Mx4(full.codes.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3),
                    full.scales.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), N)
        cache.scales[:, :, S:] = 255
        vbuf = torch.full((B, 1, cap, D + 5), float("nan"), dtype=BF, device="cuda")
        vbuf[:, :, :S, :D] = v[:, :, :S].cuda()
        qbuf = torch.full((B, H, 1, N + 7), float("nan"), dtype=qdt, device="cuda")
        qbuf[..., 3:3 + N] = q.cuda()
        want = X.decode_want(q, k.narrow(2, 0, S), v[:, :, :S])
        got = kernels.bdh_attn_decode(qbuf[..., 3:3 + N], cache.narrow(2, 0, S), vbuf[:, :, :S, :D], impl="hip")
        assert X.equal(got, want)


def ran(fn):
    ext.profile_enable(True)
    ext.profile_collect()
    try:
        out = fn()
        return out, {n for n, _ in ext.profile_collect()}
    finally:
        ext.profile_enable(False)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("kernel,shape", [("k_mx4_few", s) for s in X.FEW] + [("k_mx4_tile", s) for s in X.TILES])
def test_gemm(kernel, shape, four):
    print("gemm", kernel, shape, four, flush=True)
    a, wt, mul = X.gemm_operands(*shape, four)
    plain = X.gemm_want(a, wt, False, None)
    gated = X.gemm_want(a, wt, True, mul)
    a, wt, mul = dev(a), dev(wt), mul.cuda()
    names = set()
    for relu, m, odt, want in ((False, None, F32, plain), (False, None, BF, plain), (True, mul, BF, gated),
                               (True, mul.float(), F32, gated)):
        got, n = ran(lambda: kernels.mx4_gemm(a, wt, relu=relu, mul=m, out_dtype=odt, impl="hip"))
        names |= n
        assert X.equal(got, want)
    assert kernel in names


@pytest.mark.parametrize("M_,N,K", [(5, 70, 16424), (3, 1200, 8232), (1500, 1204, 712), (2100, 30, 16424)])
def test_gemm_in_other_memory(M_, N, K):
    """Rows off 16 bytes, shared over the heads; output rows of a token-major buffer."""
    H = 3
    a, wt, _ = X.gemm_operands(H, M_, N, K, False)
    buf = torch.full((M_, K + 5), float("nan"), dtype=BF, device="cuda")
    buf[:, 3:3 + K] = a[0].cuda()
    rows = buf[:, 3:3 + K].unsqueeze(0).expand(H, M_, K)
    o = torch.full((M_, H, N + 6), 5.0, dtype=F32, device="cuda")
    out = o[..., 3:3 + N].permute(1, 0, 2)
    kernels.mx4_gemm(rows, dev(wt), out=out, impl="hip")
    assert X.equal(out.contiguous(), X.gemm_want(a[:1].expand(H, M_, K), wt, False, None))
    assert bool((o[..., :3] == 5).all()) and bool((o[..., 3 + N:] == 5).all())
