"""Angles next to quarter turns: what is left beside the nearest one keeps its own 24 bits."""

import math

import pytest
import torch

from quashkv_amd import _native as N
from quashkv_amd.rotary import rotary

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True, scope="module")
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    N.lib()


@pytest.mark.parametrize("d", [32, 33])         # 16-byte accesses, single elements
@pytest.mark.parametrize("inverse", [False, True])
def test_next_to_quarter_turns(d, inverse):
    """Sines of e beside k quarter turns are within 10 2^-24 of themselves: e is rounded once
    (2^-24), sine and cosine are fp32's within 4 steps (8 2^-24), and rows of (1, 0) and (0, 1) add
    nothing to them.  (Beside the whole angle's fp32 the smallest of these are lost.)"""
    eps = [s << n for n in (60, 50, 44, 34, 24) for s in (1, -1, 5, -7)][:16]
    for k in range(4):
        turns = [(k * 2 ** 62 + e + 2 ** 63) % 2 ** 64 - 2 ** 63 for e in eps]
        x = torch.zeros(1, 2, d)
        x[:, 0, :16] = 1                        # head 0: (1, 0), head 1: (0, 1)
        x[:, 1, 16:32] = 1
        y, _ = rotary(x.to(DEV), None, torch.ones(1, dtype=torch.int32, device=DEV),
                      torch.tensor(turns, device=DEV), inverse=inverse)
        y = y.cpu().double()[0]
        for i, e in enumerate(eps):
            a = 2 * math.pi * e / 2 ** 64
            s, c = math.sin(a), math.cos(a)
            s, c = [(s, c), (c, -s), (-s, -c), (-c, s)][k]
            if inverse:
                s = -s
            for got, want in ((y[0, i], c), (y[0, 16 + i], s), (y[1, i], -s), (y[1, 16 + i], c)):
                assert abs(float(got) - want) <= 10 * 2.0 ** -24 * abs(want), (k, e, float(got), want)
