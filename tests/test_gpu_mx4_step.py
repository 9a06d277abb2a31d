"""The native generate step over 4-bit keys and weights in the calls around the usual one: captured and
replayed, with tables and caches in other memory, and twice at once on two streams.

All of them are the same arithmetic in the same order, so results are equal to the bit."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a ROCm GPU", allow_module_level=True)

import kernels  # noqa: E402
import mx4_oracle as M  # noqa: E402
from kernels import Mx4  # noqa: E402

BF = torch.bfloat16


class Step:
    """Inputs of a step of L layers; ``pad`` puts rows of the cache into a larger one, ``off`` the tables
    off 16 bytes."""

    def __init__(self, keys4, four, B=3, L=2, nh=4, N=512, D=256, S=37, cap=40, seed=0, pad=False, off=False):
        r = lambda *s, std=1.0: (M.rows(s, seed + len(s) + s[-1]) * std).cuda()  # noqa: E731
        self.x = r(B, D)
        w = [r(nh, N, D, std=0.1), r(nh, N, D, std=0.1).roll(1, 0), r(D, nh * N, std=0.1)]
        self.w = [kernels.mx4_quantize(t, impl="hip") for t in w] if four else [w[0].to(BF), w[1].to(BF), w[2].t().contiguous().to(BF)]
        cos, sin = kernels.rope_cos_sin(1, S, kernels.get_freqs(N).cuda())
        if off:
            cos, sin = (torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape) for t in (cos, sin))
        self.cos, self.sin = cos, sin
        rows = r(L, B, nh, cap, N)
        extra = 3 if pad else 0
        if keys4:
            q = [kernels.mx4_quantize(t, impl="hip") for t in rows]  # (four dims at a time)
            full = Mx4.empty(L, B + extra, nh, cap + extra, N, device="cuda")
            full.codes.fill_(0xA5), full.scales.fill_(0x5A)
            self.kr = full.narrow(1, extra // 2, B).narrow(3, extra // 2, cap)
            for i, t in enumerate(q):
                self.kr[i].codes.copy_(t.codes), self.kr[i].scales.copy_(t.scales)
            self.rest = [full.codes, full.scales]
        else:
            full = torch.full((L, B + extra, nh, cap + extra, N), 7.0, dtype=BF, device="cuda")
            self.kr = full.narrow(1, extra // 2, B).narrow(3, extra // 2, cap)
            self.kr.copy_(rows)
            self.rest = [full]
        self.v = r(L, B, 1, cap, D).to(BF)
        self.S = S
        self.v[0, :, 0, S] = self.x.to(BF)

    def run(self):
        out = kernels.decode_step_mx4(self.x, *self.w, self.cos, self.sin, self.kr, self.v, self.S)
        k = [t.contiguous() for t in ((self.kr.codes, self.kr.scales) if isinstance(self.kr, Mx4) else (self.kr,))]
        return [out, *k, self.v.clone()]


FORMS = [(True, False), (True, True), (False, True)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b)) and len(a) == len(b)


@pytest.mark.parametrize("keys4,four", FORMS)
@pytest.mark.parametrize("B", [3, 40])
def test_tables_and_caches_in_other_memory(keys4, four, B):
    want = Step(keys4, four, B=B).run()
    assert bool(torch.isfinite(want[0]).all())
    assert same(Step(keys4, four, B=B, off=True).run(), want)  # (RoPE in a launch of its own)
    padded = Step(keys4, four, B=B, pad=True)
    was = [t.clone() for t in padded.rest]
    assert same(padded.run(), want)
    for now, before in zip(padded.rest, was):  # one row of each (layer, sequence, head) is written, and no other
        slot = torch.zeros(now.shape[:4], dtype=torch.bool, device="cuda")
        slot[:, 1:1 + B, :, 1 + padded.S] = True
        assert torch.equal(now[~slot], before[~slot])


@pytest.mark.parametrize("keys4,four", FORMS)
def test_captured_and_replayed(keys4, four):
    steps = [Step(keys4, four, seed=1), Step(keys4, four, B=5, S=20, seed=2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in steps:
            s.run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run())
        graphs.append(g)
    for r in range(4):
        for i, s in enumerate(steps):
            s.x.copy_(M.rows(s.x.shape, 30 + r + i))
            s.v[0, :, 0, s.S] = s.x.to(BF)
        for g in (graphs if r % 2 else graphs[::-1]):
            g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for s, o in zip(steps, got):
            assert same(o, s.run())
        torch.cuda.synchronize()


@pytest.mark.parametrize("keys4,four", FORMS)
def test_two_streams_at_once(keys4, four):
    a, b = Step(keys4, four, seed=3), Step(keys4, four, B=4, seed=4)
    want = a.run(), b.run()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(one):
            x = a.run()
        with torch.cuda.stream(two):
            y = b.run()
        got.append((x, y))
    one.synchronize(), two.synchronize()
    assert all(same(x, want[0]) and same(y, want[1]) for x, y in got)
