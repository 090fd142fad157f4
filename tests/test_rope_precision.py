"""Rotary frequencies as fractions of a turn, against 60 decimal digits: what is stored is multiplied by positions of
up to 2^31, so its last bits count."""
import decimal

import numpy as np
import pytest
import torch

import vtq
from serving import TAGS, TYPES, rotation_bound, stream, within

D = decimal.Decimal
PI = D("3.14159265358979323846264338327950288419716939937510582097494459")
PLANS = [dict(theta=10000.0), dict(theta=500000.0), dict(theta=1e6), dict(theta=1.5),
         dict(theta=10000.0, scaling=vtq.ROPE_SCALE_LINEAR, factor=3.0),
         dict(theta=5e5, scaling=vtq.ROPE_SCALE_BANDS, factor=8.0, original_context=8192),
         dict(theta=1e6, scaling=vtq.ROPE_SCALE_YARN, factor=12.0, original_context=8192),
         dict(theta=10000.0, factors=[1.0 + 0.37 * i for i in range(64)])]


def _turns(rot, theta, scaling=vtq.ROPE_SCALE_NONE, factor=1.0, original_context=0, factors=None):
    """Turns a position of every pair."""
    out = []
    with decimal.localcontext() as c:
        c.prec = 60
        t, s, original = D(theta), D(factor), D(original_context)

        def index(turns):
            return rot * (original / (turns * 2 * PI)).ln() / (2 * t.ln())
        for i in range(rot // 2):
            f = (-2 * D(i) / rot * t.ln()).exp()
            if factors is not None:
                f /= D(float(np.float32(factors[i])))
            keep = D(1)
            if scaling == vtq.ROPE_SCALE_LINEAR:
                keep = D(0)
            elif scaling == vtq.ROPE_SCALE_BANDS:
                keep = (original * f / (2 * PI) - 1) / 3
            elif scaling == vtq.ROPE_SCALE_YARN:
                first, last = max(D(0), index(32).to_integral_value(decimal.ROUND_FLOOR)), min(
                    D(rot - 1), index(1).to_integral_value(decimal.ROUND_CEILING))
                keep = 1 - (i - first) / max(last - first, D(0.001))
            keep = min(D(1), max(D(0), keep))
            out.append((keep * f + (1 - keep) * f / s) / (2 * PI))
    return out


@pytest.mark.parametrize("args", PLANS)
def test_turns_are_right_to_their_last_bits(args):
    plan = vtq.Rope(128, **args).plan
    for i, want in enumerate(_turns(128, **args)):
        with decimal.localcontext() as c:
            c.prec = 60
            off = abs(D(plan.turns[i]) - (want - int(want)) * 2 ** 64)
        # cut at 2^-64, and some ten operations with 64 bits on a frequency of a sixth of a turn at most, of which
        # the exponent's error counts up to x e^-x < 0.37 times: each below 2^-64 / 6
        assert off < 4, (i, float(off))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("layout", [vtq.ROPE_HALF, vtq.ROPE_INTERLEAVED])
@pytest.mark.parametrize("args", PLANS)
def test_rotations_at_the_farthest_positions(ctx, args, layout, name):
    positions = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 12345, 2 ** 30 + 7, 10 ** 9, -10 ** 9 - 1, 10 ** 6, 0]
    rope = vtq.Rope(128, layout=layout, **args)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(len(positions), 3, 128, generator=g).to(TYPES[name])
    dx, pos = x.cuda(), torch.tensor(positions, dtype=torch.int32, device="cuda")
    y = torch.empty_like(dx)
    ctx.rope_device(rope, TAGS[name], dx.data_ptr(), 384, 128, y.data_ptr(), 384, 128, pos.data_ptr(), len(positions), 3,
                    128, stream())
    angle = torch.empty(len(positions), 64, dtype=torch.float64)
    with decimal.localcontext() as c:
        c.prec = 60
        for i, turns in enumerate(_turns(128, **args)):
            for p, position in enumerate(positions):
                whole = position * turns
                angle[p, i] = float((whole - whole.to_integral_value()) * 2 * PI)
    magnitude = float(rope.plan.magnitude)
    cos, sin = (torch.cos(angle) * magnitude)[:, None], (torch.sin(angle) * magnitude)[:, None]
    ia = torch.arange(64) if layout == vtq.ROPE_HALF else torch.arange(0, 128, 2)
    ib = ia + (64 if layout == vtq.ROPE_HALF else 1)
    want, size = torch.empty(x.shape, dtype=torch.float64), torch.empty(x.shape, dtype=torch.float64)
    a, b = x.double()[..., ia], x.double()[..., ib]
    want[..., ia], want[..., ib] = a * cos - b * sin, a * sin + b * cos
    size[..., ia], size[..., ib] = (a * cos).abs() + (b * sin).abs(), (a * sin).abs() + (b * cos).abs()
    # The angle is off by 2^31 * 4 * 2^-64 turns at most, 3e-9: a twentieth of f32's half step.  It turns (a, b), so
    # counts by their length, which is at most the sizes' sum over both rows.
    turned = 2.0 ** 31 * 4 * 2.0 ** -64 * 6.3 * magnitude
    length = torch.empty_like(size)
    length[..., ia] = length[..., ib] = (a * a + b * b).sqrt()
    within(y, want, rotation_bound(want, size, TYPES[name]) + turned * length, "y")
