"""Rotary positions (vtq_rope_device) against 64 bits."""
import numpy as np
import pytest
import torch

import vtq
from serving import TAGS, TYPES, frequencies, rotate_exact, rotation_bound, stream, within

pytestmark = pytest.mark.gpu

HALF, INTER = vtq.ROPE_HALF, vtq.ROPE_INTERLEAVED


def _rotate(ctx, rope, x, pos, y=None):
    name = next(k for k, t in TYPES.items() if t == x.dtype)
    y = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda") if y is None else y
    ctx.rope_device(rope, TAGS[name], x.data_ptr(), x.stride(0), x.stride(1), y.data_ptr(), y.stride(0), y.stride(1),
                    pos.data_ptr(), x.shape[0], x.shape[1], x.shape[2], stream())
    torch.cuda.synchronize()
    return y


def _check(ctx, x, pos, rot, layout, **scaling):
    rope = vtq.Rope(rot, layout, **scaling)
    named = dict(scaling)
    if "original_context" in named:
        named["original"] = named.pop("original_context")
    freq, magnitude = frequencies(rot, **named)
    want, size, _ = rotate_exact(x, pos, freq, magnitude, layout)
    got = _rotate(ctx, rope, x.cuda(), pos.cuda())
    within(got, want, rotation_bound(want, size, x.dtype), f"rot {rot} layout {layout} {scaling}")
    assert torch.equal(got[..., rot:].cpu(), x[..., rot:])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", [HALF, INTER])
@pytest.mark.parametrize("tokens,heads,head_dim,rot", [(1, 1, 2, 2), (1, 36, 64, 64), (8, 36, 64, 64), (3, 5, 80, 32),
                                                       (2, 7, 96, 24), (5, 3, 128, 128), (2, 2, 256, 256),
                                                       (4, 3, 100, 50), (3, 2, 77, 34), (300, 40, 128, 64),
                                                       (2, 3, 576, 64), (1, 200, 64, 20)])
def test_rotation(ctx, dtype, layout, tokens, heads, head_dim, rot):
    g = torch.Generator().manual_seed(tokens * 31 + heads * 7 + head_dim + rot)
    x = torch.randn(tokens, heads, head_dim, generator=g).to(TYPES[dtype])
    pos = torch.randint(0, 5000, (tokens,), generator=g, dtype=torch.int32)
    _check(ctx, x, pos, rot, layout)


@pytest.mark.parametrize("scaling", [
    dict(), dict(theta=1e6), dict(scaling=vtq.ROPE_SCALE_LINEAR, factor=4.0),
    dict(theta=500000.0, scaling=vtq.ROPE_SCALE_BANDS, factor=8.0, original_context=8192),
    dict(theta=500000.0, scaling=vtq.ROPE_SCALE_BANDS, factor=32.0, original_context=4096, low=2.0, high=3.0),
    dict(theta=1e6, scaling=vtq.ROPE_SCALE_YARN, factor=16.0, original_context=8192),
    dict(scaling=vtq.ROPE_SCALE_YARN, factor=2.0, original_context=2048, low=0.5, high=64.0)])
@pytest.mark.parametrize("layout", [HALF, INTER])
def test_scalings_at_near_and_far_positions(ctx, scaling, layout):
    g = torch.Generator().manual_seed(3)
    # up to a million: the 64-bit reference's own angle (2^20 turns and more, off by 2^-32) is then still good enough
    pos = torch.tensor([0, 1, 2, 63, 4095, 8191, 32768, 131071, 999999, -1, -77777], dtype=torch.int32)
    x = torch.randn(len(pos), 2, 128, generator=g)
    _check(ctx, x, pos, 128, layout, **scaling)


def test_factors_and_magnitude(ctx):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(6, 3, 64, generator=g)
    pos = torch.arange(6, dtype=torch.int32) * 1000
    factors = np.linspace(1.0, 9.0, 32).astype(np.float32)
    rope = vtq.Rope(64, HALF, factors=factors, magnitude=1.25)
    freq, _ = frequencies(64, factors=factors)
    want, size, _ = rotate_exact(x, pos, freq, 1.25, HALF)
    within(_rotate(ctx, rope, x.cuda(), pos.cuda()), want, rotation_bound(want, size, x.dtype), "factors")


def test_position_zero_and_opposite_positions(ctx):
    x = torch.randn(4, 5, 128, device="cuda")
    rope = vtq.Rope(128, HALF)
    assert torch.equal(_rotate(ctx, rope, x, torch.zeros(4, dtype=torch.int32, device="cuda")), x)
    # turning by p and by -p keeps the length of every pair and the first component of (1, 0)
    one = torch.zeros(2, 1, 128, device="cuda")
    one[:, :, :64] = 1.0
    y = _rotate(ctx, rope, one, torch.tensor([2 ** 31 - 1, -(2 ** 31 - 1)], dtype=torch.int32, device="cuda"))
    assert torch.equal(y[0, :, :64], y[1, :, :64]) and torch.equal(y[0, :, 64:], -y[1, :, 64:])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout,head_dim,rot", [(HALF, 64, 64), (INTER, 64, 32), (INTER, 76, 18), (HALF, 70, 14)])
def test_in_place_and_strided(ctx, dtype, layout, head_dim, rot):
    g = torch.Generator().manual_seed(9)
    pos = torch.randint(0, 9000, (6,), generator=g, dtype=torch.int32).cuda()
    rope = vtq.Rope(rot, layout)
    x = torch.randn(6, 5, head_dim, generator=g).to(TYPES[dtype]).cuda()
    want = _rotate(ctx, rope, x, pos)
    # in place
    z = x.clone()
    assert _rotate(ctx, rope, z, pos, y=z) is z and torch.equal(z, want)
    # heads of a packed row, heads and tokens exchanged, rows that start at odd elements
    packed = torch.full((6, 9, head_dim), 5.0, dtype=x.dtype, device="cuda")
    packed[:, 2:7] = x
    assert torch.equal(_rotate(ctx, rope, packed[:, 2:7], pos), want)
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(_rotate(ctx, rope, swapped, pos), want)
    odd = torch.full((6, 5, head_dim + 1), 5.0, dtype=x.dtype, device="cuda")
    odd[..., 1:] = x
    out = torch.full((6, 5, head_dim + 1), 5.0, dtype=x.dtype, device="cuda")
    _rotate(ctx, rope, odd[..., 1:], pos, y=out[..., 1:])
    assert torch.equal(out[..., 1:], want) and (out[..., 0] == 5.0).all()


def test_many_tokens(ctx):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(200000, 2, 8, generator=g, device="cuda")
    pos = torch.arange(200000, dtype=torch.int32, device="cuda")
    y = _rotate(ctx, vtq.Rope(8, INTER), x, pos)
    pick = torch.tensor([0, 1, 65535, 65536, 131072, 199999])
    freq, m = frequencies(8)
    want, size, _ = rotate_exact(x[pick.cuda()], pos[pick.cuda()], freq, m, INTER)
    within(y[pick.cuda()], want, rotation_bound(want, size, x.dtype), "many tokens")
