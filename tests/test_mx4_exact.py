"""The comparison of test_gpu_mx4_exact.py, on the CPU: its operands are within the bound of exact
sums, and it rejects a result that misses a key, a block of 32 elements or a pass of the query, or
counts one twice; and its shapes reach every form of the decode kernel."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import bdh_hip_ext as ext
import mx4_exact as X

F32, BF = torch.float32, torch.bfloat16


def _as(want, dtype):
    return torch.from_numpy(want).to(F32).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape", X.DECODE)
def test_decode_comparison(shape, dtype):
    _, _, Tq, S, N, D, _ = shape
    q, k, v = X.decode_operands(1, 1, Tq, S, N, D, 1, dtype, dtype)
    want = X.decode_want(q, k, v)
    assert X.equal(_as(want, dtype), want)
    qq, kv, vv = q.double().numpy()[0, 0], X.values(k)[0, 0].astype(np.float64), v.double().numpy()[0, 0]
    scores = qq @ kv.T
    wrong = []
    for j in {0, S // 2, S - 1}:  # one key missing, one twice
        term = np.outer(scores[:, j], vv[j])
        wrong += [want - term, want + term]
    nb = -(-N // 32)
    for b in {0, nb // 2, nb - 1, *range(256, nb, 256)}:  # a block of every key missing
        at = slice(32 * b, 32 * b + 32)
        wrong.append(want - (qq[:, at] @ kv[:, at].T) @ vv)
    if N > 8192:  # the passes of q after the first
        wrong.append(want - (qq[:, 8192:] @ kv[:, 8192:].T) @ vv)
    for w in wrong:
        assert not X.equal(_as(w.reshape(want.shape), dtype), want)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("shape", X.FEW + X.TILES)
def test_gemm_comparison(shape, four):
    _, m, n, K = shape
    a, wt, _ = X.gemm_operands(1, min(m, 70), min(n, 70), K, four)
    want = X.gemm_want(a, wt, False, None)
    av = (X.values(a) if four else a.float().numpy())[0]
    w = X.values(wt)[0]
    nb = -(-K // 32)
    for b in {0, nb // 2, nb - 1}:
        at = slice(32 * b, 32 * b + 32)
        for dtype in (F32, BF):
            assert not X.equal(_as(want - (av[:, at] @ w[:, at].T)[None], dtype), want)
    assert X.equal(_as(want, BF), want)


def test_decode_shapes_reach_every_form():
    """Lanes a key by the row's length, keys at a time by the chunk's (k_mx4_decode); the chunk by the
    workspace: one partial a chunk."""
    seen = set()
    for B, H, Tq, S, N, D, _ in X.DECODE:
        rows = B * H * Tq
        n = max(1, ext._lib.bdh_mx4_decode_workspace(B, H, Tq, S, N, D) // (4 * rows * D))
        chunk = next(c for c in (64, 32, 16, 8, 4) if -(-S // c) == n)
        lanes = 4 if N <= 128 else 16 if N <= 512 else 32 if N <= 1024 else 64
        each = chunk * lanes // 256
        seen.add((lanes, 1 if lanes == 4 else 4 if each >= 4 else 2 if each >= 2 and lanes == 64 else 1))
    assert seen == {(4, 1), (16, 1), (16, 4), (32, 1), (32, 4), (64, 1), (64, 2), (64, 4)}
