"""The 4-bit serving operators, as measurable cases.

Microscaled 4-bit floating point ("mx4"): a row's elements go in blocks of 32
consecutive ones (the last block of a row may be shorter); an element is a 4-bit
E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign), element 2i in the low half of
byte i, and a block has one E8M0 scale byte b that stands for 2^(b - 127).  The
scale is the smallest power of two that takes the block's largest magnitude below
7, so that it rounds to 6 at most; elements round to nearest, ties to the even
code; a block that holds an infinity or a NaN has the scale byte 255 and stands
for NaN.

* ``quantize``: rows to mx4 and back to the values they stand for, as weights are
  laid out for serving and as a chunked prefill reads the cache back.
* ``rope``: the RoPE of latent rows (fp32 products and sum) into the 4-bit slots of
  a KV cache, and rounded once as the decode's query rows.
* ``decode``: one query a head against the keys of a 4-bit cache,
  out = (q K^T) V: BDH's attention has no softmax and no scale.
* ``gemm``: the dense products of a layer with 4-bit weights, out = [mul *] [relu]
  (a wt^T), a in bf16 or itself in mx4.

Sizes are those of the repository's configurations (n_embd 256, 4 heads of 8192
latents; the batches and lengths of ``bench.py`` and ``perf/cases.py``), or generic.

The ranges (``draw``): batch 1 to 64, heads 1 to 8, latent widths 16 to 16384 with
ragged last blocks, 1 to 16384 cached rows, 1 to 2048 new rows, products of 1 to
8192 rows, 16 to 32768 wide and to 65536 deep, fp32 and bf16, contiguous and permuted rows,
packed and capacity-strided caches.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _kernels():
    pkg = str(Path.cwd() / "bdh-gpu-fast_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import kernels

    return kernels


# ------------------------------------------------------------------- cases
def listed():
    return [
        # A model's encoder, fp32 parameters, laid out for serving.
        dict(name="quantize_weights_fp32", op="quantize", B=1, nh=4, T=8192, N=256, dtype="fp32", permuted=False),
        # The latents of ragged documents, read in the model's (B, T, nh, N) memory.
        dict(name="quantize_latent_bf16", op="quantize", B=6, nh=4, T=777, N=8192, dtype="bf16", permuted=True),
        # A generate step's new row of a few sequences: the smallest call (launches and latency).
        dict(name="rope_step_bf16", op="rope", B=8, nh=4, T=1, S=300, cap=512, N=8192, dtype="bf16", q=True),
        # A batch's prompts into the cache: the fused attention rotates for itself, so only the slots are written.
        dict(name="rope_prefill_bf16", op="rope", B=8, nh=4, T=512, S=0, cap=768, N=8192, dtype="bf16", q=False),
        # A chunk after a cached past, without autocast, latents of a width that ends inside a block.
        dict(name="rope_chunk_fp32", op="rope", B=3, nh=2, T=137, S=190, cap=512, N=1000, dtype="fp32", q=True),
        # A batched generate step late in the sequence.
        dict(name="decode_batch_bf16", op="decode", B=64, nh=4, S=511, cap=512, N=8192, D=256, dtype="bf16"),
        # Interactive generate without autocast: one sequence, fp32 query and values.
        dict(name="decode_single_fp32", op="decode", B=1, nh=4, S=301, cap=1024, N=8192, D=256, dtype="fp32"),
        # Long documents, as many bytes of keys as the batch: two sequences in a cache with room to go on.
        dict(name="decode_long_bf16", op="decode", B=2, nh=4, S=16001, cap=16384, N=8192, D=256, dtype="bf16"),
        # encoder_v of a generate step: a product a head for 8 sequences, ReLU and the gate with the latent.
        dict(name="gemm_gate_step", op="gemm", H=4, M=8, N=8192, K=256, a="bf16", relu=True, mul=True, out="bf16"),
        # The decoder of the same step: few rows, a deep contraction.
        dict(name="gemm_decoder_step", op="gemm", H=1, M=8, N=256, K=32768, a="bf16", relu=False, mul=False, out="fp32"),
        # The decoder of a prefill over ragged documents (8 of 777 tokens).
        dict(name="gemm_decoder_prefill", op="gemm", H=1, M=6216, N=256, K=32768, a="bf16", relu=False, mul=False,
             out="bf16"),
        # Both operands in 4 bits, a large square-like product.
        dict(name="gemm_mx4_both", op="gemm", H=1, M=4096, N=8192, K=8192, a="mx4", relu=False, mul=False, out="bf16"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: an operator, then sizes over its range, spread by logarithm."""
    op = rng.choice(["quantize", "rope", "rope", "decode", "decode", "decode", "gemm", "gemm", "gemm"])
    for _ in range(1000):
        nh = rng.choice([1, 2, 4, 8])
        N = _logint(rng, 16, 16384)
        N = rng.choice([N, -(-N // 32) * 32, -(-N // 256) * 256, 8192])
        dt = rng.choice(["fp32", "bf16", "bf16"])
        B = _logint(rng, 1, 64)
        if op == "quantize":
            c = dict(op=op, B=B, nh=nh, T=_logint(rng, 1, 2048), N=N, dtype=dt, permuted=rng.choice([True, False]))
        elif op == "rope":
            T, S = rng.choice([1, _logint(rng, 1, 2048)]), _logint(rng, 1, 1024)
            c = dict(op=op, B=B, nh=nh, T=T, S=S, cap=S + T + rng.randrange(0, 65), N=N + N % 2, dtype=dt,
                     q=rng.choice([True, False]))
        elif op == "decode":
            S = _logint(rng, 1, 16384)
            c = dict(op=op, B=B, nh=nh, S=S, cap=S + rng.randrange(0, 65), N=N,
                     D=rng.choice([32, 64, 96, 128, 192, 256, 256, 384, 512]), dtype=dt)
        else:
            few = rng.choice([True, False])
            c = dict(op=op, H=rng.choice([1, 1, 2, 4]), M=_logint(rng, 1, 64) if few else _logint(rng, 64, 8192),
                     N=rng.choice([_logint(rng, 16, 32768), 256, 8192]), K=rng.choice([N, 256, 512, 2 * N]),
                     a=rng.choice(["bf16", "bf16", "mx4"]), relu=rng.choice([True, False]),
                     mul=rng.choice([True, False]), out=rng.choice(["bf16", "fp32"]))
        w = work(c)
        if w["bytes"] <= 6e8 and w["flops"] <= 5.4e11:
            return c
    raise RuntimeError("no case drawn")


# ------------------------------------------------------------------ inputs
def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _rotated(g, rows, N):
    """Rows as a cache holds them: ReLU latents, about half zeros, each pair turned by some angle."""
    x = torch.relu(_randn(g, rows, N + N % 2, std=0.32)).view(rows, -1, 2)
    ph = torch.rand(rows, x.size(1), generator=g, device="cuda") * (2 * math.pi)
    c, s = torch.cos(ph), torch.sin(ph)
    return torch.stack((x[..., 0] * c - x[..., 1] * s, x[..., 1] * c + x[..., 0] * s), -1).flatten(1)[:, :N]


def _pack(x):
    """fp32 rows (R, N) in mx4: codes (R, 16 ceil(N / 32)) and scale bytes (R, ceil(N / 32))."""
    y, b = _scaled(x)
    i = _index(y.abs()) + 8 * (y < 0)
    i = i.to(torch.uint8).flatten(1)
    return i[:, 0::2] + 16 * i[:, 1::2], b.to(torch.uint8)


def _packed(c, g, rows, N, make):
    """mx4 rows in pieces, so that a large cache needs no fp32 copy of itself."""
    kb = -(-N // 32)
    codes = torch.empty(rows, 16 * kb, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, kb, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // N)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        codes[r:r + n], scales[r:r + n] = _pack(make(g, n, N))
    return codes, scales


def _gauss(g, rows, N):
    return _randn(g, rows, N, std=0.02)


def _acts(g, rows, N):
    return _randn(g, rows, N)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"case": c}
    op = c["op"]
    if op in ("quantize", "rope"):
        B, nh, T, N, dt = c["B"], c["nh"], c["T"], c["N"], _DTYPES[c["dtype"]]
        if op == "quantize" and not c["permuted"]:
            s["x"] = _randn(g, B, nh, T, N, std=0.02).to(dt)
        else:  # the latent, in the model's memory
            s["x"] = torch.relu(_randn(g, B, T, nh, N, std=0.32)).to(dt).permute(0, 2, 1, 3)
        if op == "rope":
            kb = -(-N // 32)
            m = torch.arange(N, device="cuda", dtype=torch.float64)
            f = (1.0 / (65536.0 ** ((m / 2).floor() * 2 / N)) / (2 * math.pi)).float()
            ph = (torch.arange(c["S"], c["S"] + T, device="cuda").float()[:, None] * f % 1) * (2 * math.pi)
            s["cos"], s["sin"] = torch.cos(ph).view(1, 1, T, N), torch.sin(ph).view(1, 1, T, N)
            s["codes"] = torch.zeros(B, nh, c["cap"], 16 * kb, dtype=torch.uint8, device="cuda")
            s["scales"] = torch.zeros(B, nh, c["cap"], kb, dtype=torch.uint8, device="cuda")
    elif op == "decode":
        B, nh, N, D, dt = c["B"], c["nh"], c["N"], c["D"], _DTYPES[c["dtype"]]
        codes, scales = _packed(c, g, B * nh * c["cap"], N, _rotated)
        s["codes"] = codes.view(B, nh, c["cap"], -1).narrow(2, 0, c["S"])
        s["scales"] = scales.view(B, nh, c["cap"], -1).narrow(2, 0, c["S"])
        s["v"] = _randn(g, B, 1, c["cap"], D).to(dt).narrow(2, 0, c["S"])
        s["q"] = _rotated(g, B * nh, N).to(dt).contiguous().view(B, nh, 1, N)
    else:
        H, M, N, K = c["H"], c["M"], c["N"], c["K"]
        s["w"], s["ws"] = (t.view(H, N, -1) for t in _packed(c, g, H * N, K, _gauss))
        if c["a"] == "mx4":
            s["a"], s["as"] = (t.view(H, M, -1) for t in _packed(c, g, H * M, K, _acts))
        else:
            s["a"] = _randn(g, H, M, K).to(torch.bfloat16)
        if c["mul"]:  # the latent, token-major
            s["mul"] = torch.relu(_randn(g, M, H, N, std=0.32)).to(torch.bfloat16).permute(1, 0, 2)
    return s


# --------------------------------------------------------------------- run
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _scaled(x):
    """fp32 rows (..., N) in blocks (..., ceil(N / 32), 32), divided by their scales, and the scale bytes."""
    pad = -x.size(-1) % 32
    if pad:
        x = torch.cat((x, x.new_zeros(*x.shape[:-1], pad)), -1)
    x = x.view(*x.shape[:-1], -1, 32)
    m, e = torch.frexp(x.abs().amax(-1))  # the largest is m 2^e, 0.5 <= m < 1
    e = (e - 3 + (m >= 0.875).int()).clamp(-127, 127)
    return torch.ldexp(x, -e.unsqueeze(-1)), e + 127


def _index(y):
    """The code of a magnitude: nearest, ties to even."""
    i = torch.where(y < 2, torch.round(2 * y), torch.where(y < 4, torch.round(y) + 2, torch.round(y / 2) + 4))
    return i.clamp_max(7).to(torch.int32)


def _grid(device, dtype=torch.float32):
    return torch.tensor(_GRID + tuple(-v for v in _GRID), device=device, dtype=dtype)


def _round4(x):
    """The values that fp32 rows stand for in mx4."""
    y, b = _scaled(x)
    v = torch.ldexp(_grid(x.device)[_index(y.abs())], (b - 127).unsqueeze(-1))
    return (v * torch.sign(y)).flatten(-2)[..., : x.size(-1)]


def _values(codes, scales, N):
    """fp32 values of mx4 rows."""
    lut = _grid(codes.device)
    v = torch.stack((lut[(codes & 15).int()], lut[(codes >> 4).int()]), -1)
    v = v.view(*codes.shape[:-1], -1, 32) * torch.exp2(scales.float() - 127).unsqueeze(-1)
    return v.flatten(-2)[..., :N]


def _run_plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "quantize":
        return _round4(s["x"].float()).to(torch.bfloat16)
    if op == "rope":
        x, cos, sin = s["x"].float(), s["cos"], s["sin"]
        x0, x1 = x[..., 0::2], x[..., 1::2]
        y0 = x0 * cos[..., 0::2] - x1 * sin[..., 0::2]
        y1 = x1 * cos[..., 1::2] + x0 * sin[..., 1::2]
        r = torch.stack((y0, y1), -1).flatten(-2)
        slots = _round4(r).to(torch.bfloat16)
        return (slots, r.to(s["x"].dtype)) if c["q"] else slots
    if op == "decode":
        k = _values(s["codes"], s["scales"], c["N"])
        sc = torch.matmul(k, s["q"].float().transpose(2, 3).contiguous()).squeeze(-1)  # (B, nh, S)
        return torch.matmul(sc, s["v"][:, 0].float()).unsqueeze(2).to(s["q"].dtype)
    w = _values(s["w"], s["ws"], c["K"]).transpose(1, 2).contiguous()
    a = _values(s["a"], s["as"], c["K"]) if c["a"] == "mx4" else s["a"].float()
    y = torch.matmul(a, w)
    if c["relu"]:
        y = torch.relu(y)
    if c["mul"]:
        y = y * s["mul"].float()
    return y.to(_DTYPES[c["out"]])


def run(s):
    if not own:
        return _run_plain(s)
    kernels = _kernels()
    c, op = s["case"], s["case"]["op"]
    if op == "quantize":
        return kernels.mx4_dequantize(kernels.mx4_quantize(s["x"], impl="hip"), torch.bfloat16, impl="hip")
    if op == "rope":
        slot = kernels.Mx4(s["codes"], s["scales"], c["N"]).narrow(2, c["S"], c["T"])
        r = torch.empty(s["x"].shape, dtype=s["x"].dtype, device="cuda") if c["q"] else None
        kernels.mx4_rope(s["x"], s["cos"], s["sin"], slot, out=r, impl="hip")
        values = kernels.mx4_dequantize(slot, torch.bfloat16, impl="hip")
        return (values, r) if c["q"] else values
    if op == "decode":
        past = kernels.Mx4(s["codes"], s["scales"], c["N"])
        return kernels.bdh_attn_decode(s["q"], past, s["v"], impl="hip")
    wt = kernels.Mx4(s["w"], s["ws"], c["K"])
    a = kernels.Mx4(s["a"], s["as"], c["K"]) if c["a"] == "mx4" else s["a"]
    return kernels.mx4_gemm(a, wt, relu=c["relu"], mul=s.get("mul"), out_dtype=_DTYPES[c["out"]], impl="hip")


# -------------------------------------------------------------------- work
def work(case):
    c, op = case, case["op"]
    if op in ("quantize", "rope"):
        B, nh, T, N, e = c["B"], c["nh"], c["T"], c["N"], 2 if c["dtype"] == "bf16" else 4
        n, rows = B * nh * T * N, B * nh * T
        b = e * n + 2 * rows * 17 * -(-N // 32) + 2 * n  # rows in, their 4-bit form out and in again, its values out
        if op == "rope":
            b += 2 * 4 * T * N + (e * n if c["q"] else 0)
        return {"bytes": b, "flops": (6 if op == "rope" else 3) * n}
    if op == "decode":
        B, nh, S, N, D, e = c["B"], c["nh"], c["S"], c["N"], c["D"], 2 if c["dtype"] == "bf16" else 4
        return {"flops": 2 * B * nh * S * (N + D),
                "bytes": 17 * -(-N // 32) * B * nh * S + e * (B * S * D + B * nh * (N + D))}
    H, M, N, K = c["H"], c["M"], c["N"], c["K"]
    a = 17 * -(-K // 32) * M if c["a"] == "mx4" else 2 * M * K
    return {"flops": 2 * H * M * N * K,
            "bytes": H * (a + 17 * -(-K // 32) * N + M * N * ((4 if c["out"] == "fp32" else 2) + (2 if c["mul"] else 0)))}


# ------------------------------------------------------------------- exact
def _exact_round4(x):
    """Values in mx4 of float64 rows that hold fp32 values: the definition, by its borders."""
    n = x.size(-1)
    out = torch.zeros_like(x)
    # ties to the even code: a border belongs to its upper neighbour where that one's index is even
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    up = torch.tensor([False, True, False, True, False, True, False], device=x.device)
    borders = torch.where(up, torch.nextafter(mid, torch.zeros_like(mid)), mid)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    for k in range(0, n, 32 * 64):  # some blocks at a time
        part = x[..., k:k + 32 * 64]
        short = -part.size(-1) % 32
        blocks = torch.nn.functional.pad(part, (0, short)).unflatten(-1, (-1, 32))
        top = blocks.abs().amax(-1, keepdim=True)
        p = torch.ceil(torch.log2(torch.clamp_min(top, 2.0 ** -140) / 7.0))
        p = torch.where(top * torch.exp2(-p) >= 7.0, p + 1, p)
        p = torch.where(top * torch.exp2(-p) < 3.5, p - 1, p).clamp(-127, 127)
        i = torch.bucketize((blocks * torch.exp2(-p)).abs().contiguous(), borders)
        v = torch.copysign(grid[i], blocks) * torch.exp2(p)
        out[..., k:k + 32 * 64] = v.flatten(-2)[..., : part.size(-1)]
    return out


def _exact_values(codes, scales, N):
    """float64 values of mx4 rows, from the bits: sign, two exponent bits, one of mantissa."""
    nib = torch.stack((codes % 16, codes // 16), -1).flatten(-2).to(torch.int64)
    e, m = (nib >> 1) & 3, (nib & 1).double()
    mag = torch.where(e == 0, 0.5 * m, torch.exp2((e - 1).double()) * (1 + 0.5 * m))
    v = torch.where(nib >= 8, -mag, mag).unflatten(-1, (-1, 32))
    return (v * torch.exp2(scales.double() - 127).unsqueeze(-1)).flatten(-2)[..., :N]


def exact(case, seed):
    s = prepare(case, seed)
    c, op = s["case"], s["case"]["op"]
    if op == "quantize":
        return torch.cat([_exact_round4(x.double()) for x in s["x"].split(1)])
    if op == "rope":
        # products and their sum are rounded to fp32 by the definition (of two fp32 numbers the
        # float64 product is exact, and so is the double rounding of their sum)
        cos, sin = s["cos"].double(), s["sin"].double()
        slots, rows = [], []
        for x in s["x"].split(1):
            x = x.double()
            r = torch.empty_like(x)
            a = [(x[..., i::2] * t[..., j::2]).float().double()
                 for i, t, j in ((0, cos, 0), (1, sin, 0), (1, cos, 1), (0, sin, 1))]
            r[..., 0::2] = (a[0] - a[1]).float()
            r[..., 1::2] = (a[2] + a[3]).float()
            slots.append(_exact_round4(r))
            rows.append(r)
        return (torch.cat(slots), torch.cat(rows)) if c["q"] else torch.cat(slots)
    if op == "decode":
        B, nh, S, N, D = c["B"], c["nh"], c["S"], c["N"], c["D"]
        out = torch.zeros(B, nh, 1, D, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 27) // N)
        for b in range(B):
            for h in range(nh):
                for r in range(0, S, step):
                    k = _exact_values(s["codes"][b, h, r:r + step], s["scales"][b, h, r:r + step], N)
                    out[b, h, 0] += (k @ s["q"][b, h, 0].double()) @ s["v"][b, 0, r:r + step].double()
        return out
    H, M, N, K = c["H"], c["M"], c["N"], c["K"]
    out = torch.empty(H, M, N, dtype=torch.float64, device="cuda")
    for h in range(H):
        a = _exact_values(s["a"][h], s["as"][h], K) if c["a"] == "mx4" else s["a"][h].double()
        for n in range(0, N, 4096):
            w = _exact_values(s["w"][h, n:n + 4096], s["ws"][h, n:n + 4096], K)
            out[h, :, n:n + 4096] = a @ w.t()
    if c["relu"]:
        out = out.clamp_min(0)
    return out * s["mul"].double() if c["mul"] else out
