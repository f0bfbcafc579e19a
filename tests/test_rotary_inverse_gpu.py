"""Turning back, in every type, and positions at the ends of their types: against the plan's own turns in whole numbers.

f = 2^-24; the tolerance is test_decode_gpu.py's: 8 f of a pair's size and one rounding to the type."""
import math

import pytest
import torch

from tts_amd import ops

from .test_decode_gpu import F, TYPES, _g, _within, u

pytestmark = pytest.mark.gpu


def _turned(x, positions, plan, inverse):
    """x in 64 bits by positions * turns modulo 2^64, exactly, as a fraction of a circle."""
    turns = plan.turns.cpu().tolist()
    phase = torch.tensor([[((-p if inverse else p) * t % 2 ** 64) / 2.0 ** 64 for t in turns] for p in positions], dtype=torch.float64)
    rd = plan.rotary_dim
    c, s = (plan.amplitude * f(2 * math.pi * phase)[:, None] for f in (torch.cos, torch.sin))
    one, two = (slice(0, rd, 2), slice(1, rd, 2)) if plan.interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    out, pair = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    a, b = x.double()[..., one], x.double()[..., two]
    out[..., one], out[..., two] = a * c - b * s, b * c + a * s
    pair[..., one] = pair[..., two] = plan.amplitude * (a.abs() + b.abs())
    return out, pair


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,dim,rd,inter,scaling", [(3, 64, 64, False, None), (2, 80, 40, True, {"kind": "linear", "factor": 4.0}), (1, 66, 34, False, None),
                                                        (5, 128, 64, True, {"kind": "ramp", "factor": 8.0, "trained_len": 4096})])
def test_back_and_at_the_ends(gpu, dtype, heads, dim, rd, inter, scaling):
    plan = ops.Rotary(dim, rd, interleaved=inter, scaling=scaling, device=gpu)
    for kind, values in ((torch.int64, [0, 1, -1, 77, 2 ** 31, -2 ** 31 - 1, 2 ** 40 + 3, 2 ** 63 - 1, -2 ** 63]), (torch.int32, [0, 5, -5, 2 ** 31 - 1, -2 ** 31])):
        x = torch.randn(len(values), heads, dim, generator=_g(dim)).to(dtype)
        pos = torch.tensor(values, dtype=kind, device=gpu)
        for inverse in (False, True):
            got = ops.rotary(plan, x.to(gpu), pos, inverse=inverse)
            want, pair = _turned(x, values, plan, inverse)
            _within(got, want, u(dtype) * want.abs() * (1 + 8 * F) + 8 * F * pair + torch.finfo(dtype).tiny, "%s %s" % (kind, inverse))
            assert torch.equal(got[..., rd:].cpu(), x[..., rd:])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_there_and_back_is_where_it_was(gpu, dtype):
    """Without an amplitude the turn back undoes the turn, but for a rounding to the type on the way and one at the end: u (|a| + |b|) each."""
    plan = ops.Rotary(64, device=gpu)
    x = torch.randn(50, 3, 64, generator=_g(4)).to(dtype)
    pos = torch.arange(50, device=gpu) * 977 - 1000
    back = ops.rotary(plan, ops.rotary(plan, x.to(gpu), pos), pos, inverse=True)
    size = x.double().abs()
    pair = torch.cat([size[..., :32] + size[..., 32:]] * 2, -1)
    _within(back, x.double(), (2 * u(dtype) + 24 * F) * pair + torch.finfo(dtype).tiny)
