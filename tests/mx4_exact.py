"""Operands of the 4-bit products whose sums fp32 holds exactly, in any order.

Factors are small whole numbers, key and weight rows E2M1 codes under the scales 1/2, 1 and 2: a
product is a multiple of 1/4, and where the sum of all magnitudes stays below 2^22 (2^24 quarters)
every partial sum of every order is exact.  So is the result, but for its one rounding to bf16: a
result has to be equal, and one that misses a key, a block or a pass, or counts one twice, is not.
"""

from __future__ import annotations

import numpy as np
import torch

import mx4_oracle as M
from kernels import Mx4

BF = torch.bfloat16
MOST = 2.0 ** 22


def ints(shape, seed: int, top: int, dtype=torch.float32) -> torch.Tensor:
    g = torch.Generator("cpu").manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g).to(dtype)


def rows4(shape, seed: int) -> Mx4:
    """Random codes, a block's scale 1/2, 1 or 2; zeros behind a row's end."""
    g = torch.Generator("cpu").manual_seed(seed)
    n, kb = shape[-1], -(-shape[-1] // 32)
    nib = torch.randint(0, 16, (*shape[:-1], 32 * kb), generator=g, dtype=torch.uint8)
    nib[..., n:] = 0
    return Mx4(nib[..., 0::2] + 16 * nib[..., 1::2],
               torch.randint(126, 129, (*shape[:-1], kb), generator=g, dtype=torch.uint8), n)


def values(m: Mx4) -> np.ndarray:
    """float32 values (exact), an outer row at a time."""
    out = np.empty(m.shape, np.float32)
    for i in np.ndindex(*m.shape[:-2]):
        out[i] = M.values(Mx4(m.codes[i], m.scales[i], m.width))
    return out


def decode_operands(B, H, Tq, S, N, D, hv, qdt, vdt):
    """q, k, v on the host: v of -1, 0, 1; in fp32 a query has values that bf16 does not hold."""
    q = ints((B, H, Tq, N), 1, 2)
    if qdt == torch.float32:
        q[..., ::592] *= 257
    return q.to(qdt), rows4((B, H, S, N), 2), ints((B, hv, S, D), 3, 1, vdt)


def decode_want(q, k, v) -> np.ndarray:
    """float64, from operands within the bound."""
    qq, vv, kv = q.double().numpy(), v.double().numpy(), values(k)
    B, H, Tq, _ = qq.shape
    out = np.zeros((B, H, Tq, vv.shape[-1]))
    for b in range(B):
        for h in range(H):
            s = qq[b, h] @ kv[b, h].T.astype(np.float64)
            assert (np.abs(qq[b, h]) @ np.abs(kv[b, h]).T).max(initial=0) < MOST
            vh = vv[b, h if v.size(1) > 1 else 0]
            assert (np.abs(s) @ np.abs(vh)).max(initial=0) < MOST
            out[b, h] = s @ vh
    return out


def gemm_operands(H, M_, N, K, four, mul_dtype=BF):
    a = rows4((H, M_, K), 1) if four else ints((H, M_, K), 1, 2, BF)
    return a, rows4((H, N, K), 2), ints((M_, H, N), 3, 1, mul_dtype).permute(1, 0, 2)


def gemm_want(a, wt, relu: bool, mul) -> np.ndarray:
    av = values(a) if isinstance(a, Mx4) else a.float().numpy()
    w = values(wt)
    # (a magnitude of wt is 12 at most: the bound, without another product)
    assert 12 * np.abs(av).sum(-1, dtype=np.float64).max(initial=0) < MOST
    out = np.stack([x @ y.T for x, y in zip(av, w)]).astype(np.float64)  # exact in fp32, in any order
    out = np.maximum(out, 0) if relu else out
    return out if mul is None else out * mul.double().numpy()


def equal(got: torch.Tensor, want: np.ndarray) -> bool:
    """Whether ``got`` is ``want``, rounded once to its type."""
    w = torch.from_numpy(np.ascontiguousarray(want)).to(torch.float32)
    assert bool((w.double() == torch.from_numpy(want)).all())
    return got.shape == w.shape and torch.equal(got.cpu(), w.to(got.dtype))


# (B, H, Tq, S, N, D, value heads): the decode kernel's lanes a key and keys at a time, its loops of
# several pieces and their rests, passes of q, last chunks and groups that are not full
DECODE = [
    (32, 4, 1, 130, 8192, 64, 1), (16, 4, 1, 100, 8192, 64, 1), (64, 4, 1, 70, 8224, 64, 1), (40, 4, 1, 130, 2080, 256, 1),
    (24, 4, 1, 131, 6200, 48, 4), (24, 4, 1, 131, 4992, 64, 1), (2, 4, 1, 301, 8192, 256, 1), (1, 2, 1, 9, 20001, 512, 1),
    (1, 1, 2, 19, 8224, 64, 1), (40, 4, 2, 67, 16416, 40, 1), (12, 2, 3, 35, 16384, 128, 2), (1, 2, 1, 1203, 4096, 64, 1),
    (64, 4, 1, 70, 1000, 64, 1), (3, 4, 1, 90, 1024, 32, 4), (64, 4, 1, 150, 500, 64, 1), (2, 4, 1, 333, 512, 64, 1),
    (64, 4, 1, 200, 128, 64, 1), (1, 1, 1, 2100, 96, 33, 1),
]

FEW = [  # (H, M, N, K): few rows; waves a tile, splits, K that ends inside a load of eight blocks, several tiles
    (1, 8, 256, 32768), (4, 8, 512, 256), (1, 31, 33, 16416), (1, 5, 40, 16384), (2, 3, 300, 20001), (1, 64, 200, 33),
    (1, 33, 31, 8200), (3, 3, 1024, 2000), (1, 20, 2052, 13504), (1, 1, 70, 32800), (2, 3, 300, 600), (1, 8, 256, 1100),
]

TILES = [  # (H, M, N, K): many rows; both tile heights and stages, one column of tiles, K in splits, ragged all round
    (1, 2049, 2047, 2000), (2, 1100, 1000, 2080), (1, 6000, 200, 3200), (1, 4090, 4000, 520), (1, 3100, 17, 32800),
    (1, 5000, 250, 8224), (3, 900, 1501, 1111), (1, 8000, 1000, 300), (1, 700, 300, 16448), (1, 6216, 256, 4096),
    (1, 6000, 200, 3264), (1, 33000, 250, 576), (1, 2500, 1500, 8256),
]
