"""Attention's softmax weights where rounding shows most: maxima that rise late at large scores, and keys whose
weights are far below the largest one.  Scores are chosen so that they are exact in f32."""
import math

import numpy as np
import pytest
import torch

import vtq
from serving import F32_HALF_STEP, TAGS, TYPES, half_step, smallest, stream, within
from vtq import probe

pytestmark = pytest.mark.gpu
U = F32_HALF_STEP


def _attend(ctx, name, cache, q, k, v, heads, lens, pages, page, prefix=0, live=None, one_range=False, shared=None,
            scale=1.0):
    """k, v [n_pages, kv_heads, page, head_dim]; a token each of len(lens) sequences, the first `live` of the call's
    tokens; the others only choose how the work is split."""
    kv_heads, d, tokens = k.shape[1], k.shape[3], q.shape[0]
    live = len(lens) if live is None else live
    lists = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in
             (list(range(len(lens) + 1)), lens, pages, [0] * max(1, -(-prefix // page)))]
    c = vtq.KvCache(TAGS[cache], k.data_ptr(), v.data_ptr(), k.shape[0], page, kv_heads, d)
    b = vtq.KvBatch(len(lens), lists[0].data_ptr(), lists[1].data_ptr(), lists[2].data_ptr(), len(pages[0]),
                    max_q=tokens if tokens > len(lens) else 1, prefix_len=prefix,
                    prefix_pages=lists[3].data_ptr() if prefix else None)
    plan = probe.attention_plan(c, b, TAGS[name], tokens, heads)
    if one_range:
        assert plan["own_splits"] == 1 and plan["prefix_splits"] == 0
    if shared is not None:
        assert plan["shared_own"] == shared
    need = ctx.attention_workspace(c, b, TAGS[name], tokens, heads)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    y = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    ctx.attention_device(c, b, TAGS[name], tokens, heads, q.data_ptr(), q.stride(0), q.stride(1), y.data_ptr(),
                         y.stride(0), y.stride(1), scale, ws.data_ptr(), need, stream(), lse_ptr=lse.data_ptr())
    torch.cuda.synchronize()
    return y[:live].double().cpu(), lse[:live].double().cpu()


def _queries(tokens, heads, d, name, *first):
    q = torch.zeros(tokens, heads, d)
    for i, x in enumerate(first):
        q[..., i] = x
    q = q.to(TYPES[name])
    assert [float(x) for x in q[0, 0, :len(first)]] == list(first)
    return q.cuda()


@pytest.mark.parametrize("name,cache", [("f32", "f32"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shared", [True, False])
def test_a_late_maximum_keeps_the_earlier_weights(ctx, name, cache, d, shared):
    # 256 keys with a score S of some 2^18, then four that are higher by 6, one in every tile of a wave: weights 1 and
    # e^6.  S log2(e) in f32 is off by up to 2^-6, which must cancel.
    c = float(np.float32(1.44269504088896340736))
    k0 = max(range(200, 257), key=lambda x: abs(1024 * x * c - float(np.float32(1024 * x * c))))
    lost = abs(1024 * k0 * c - float(np.float32(1024 * k0 * c)))
    assert lost > 0.01  # of a power of two
    n, high = 353, torch.tensor([256, 288, 320, 352])
    kv_heads, batch = (1, 1) if shared else (8, 64)
    heads = 64 if shared else 8
    k = torch.zeros(1, kv_heads, 512, d)
    k[..., 0] = k0
    k[:, :, high, 1] = 6.0
    v = torch.ones(1, kv_heads, 512, d)
    v[:, :, high] = -1.0
    q = _queries(1024 if shared else batch, heads, d, name, 1024.0, 1.0)
    y, lse = _attend(ctx, name, cache, q, k.to(TYPES[cache]).cuda(), v.to(TYPES[cache]).cuda(), heads, [n] * batch,
                     [[0]] * batch, 512, one_range=True, shared=shared)
    low, top = float(n - 4), 4 * math.exp(6.0)
    want = torch.full(y.shape, (low - top) / (low + top), dtype=torch.float64)
    # Differences of 6 times log2(e), which is off by u, and the exponential by 4 u: 6 * 1.45 * 2 u + 4 u; weights are off
    # by twice that, sums by a u a key; weights and the result round to the type.  (Twice: values of both signs.)
    rel = 2.1 * (6 * 1.45 * 2 * U + 4 * U) + n * U + (0 if name == "f32" else half_step(q.dtype) * 1.01)
    bound = rel + half_step(q.dtype) * want.abs() * 1.01 + smallest(q.dtype)
    # what the lost part of a power of two would do to the 256 keys before the first rise, is more than that
    assert lost * math.log(2) * 2 * 256 * top / (low + top) ** 2 > 1.2 * float(bound[0, 0, 0])
    within(y, want, bound, "y")
    want_l = torch.full(lse.shape, 1024.0 * k0 + math.log(low + top), dtype=torch.float64)
    within(lse, want_l, 4 * U * want_l + rel, "lse")


# heads, KV heads, tokens of the call, sequences, own keys, prefix: a wave's own rows and tiles of its own, with and
# without parts, and the prefix
SHAPES = [(64, 1, 1024, 1, 500, 0), (64, 1, 1, 1, 500, 0), (8, 8, 64, 64, 500, 0), (4, 1, 1, 1, 500, 0),
          (4, 2, 20, 20, 32, 500), (2, 1, 1, 1, 32, 500)]


@pytest.mark.parametrize("name,cache", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"),
                                        ("f32", "bf16")])
@pytest.mark.parametrize("scale", [3.0e7, 1.1e10, 1.3e20, 1.0e30])
@pytest.mark.parametrize("heads,kv_heads,tokens,batch,n,prefix", SHAPES)
def test_scores_of_any_size_in_f32(ctx, heads, kv_heads, tokens, batch, n, prefix, scale, name, cache):
    # products of -7 to 5 times a large scale: the keys of 5 share the weight, the others, 3e7 and more below, have none
    g = torch.Generator().manual_seed(n + prefix)
    k = torch.zeros(2, kv_heads, 512, 64)
    k[..., 0] = torch.randint(-7, 5, (2, kv_heads, 512), generator=g).float()
    for page, place in ((0, 40), (0, 41), (0, 333), (1, 3), (1, 30), (1, 200), (1, 497)):
        k[page, :, place, 0] = 5.0
    v = torch.randn(2, kv_heads, 512, 64, generator=g).to(TYPES[cache])
    q = _queries(tokens, heads, 64, name, 1.0)
    y, lse = _attend(ctx, name, cache, q, k.to(TYPES[cache]).cuda(), v.cuda(), heads, [n] * batch, [[1]] * batch, 512,
                     prefix=prefix, live=min(tokens, batch), scale=scale)
    ks, vs = (torch.cat([x[0, :, :prefix], x[1, :, :n]], 1).double() for x in (k, v))
    has = (ks[..., 0] == 5.0).double()[..., None]
    count = has.sum(1)
    want = ((has * vs).sum(1) / count).repeat_interleave(heads // kv_heads, 0).expand(y.shape)
    size = ((has * vs.abs()).sum(1) / count).repeat_interleave(heads // kv_heads, 0).expand(y.shape)
    # weights of 1, at most 7 of them: sums and the quotient round in f32, then the result to its type
    within(y, want, 10 * U * size + half_step(q.dtype) * want.abs() * 1.01 + smallest(q.dtype), "y")
    f32_scale = float(torch.tensor(scale))
    want_l = (5.0 * f32_scale + count.log()).squeeze(-1).repeat_interleave(heads // kv_heads).expand(lse.shape)
    within(lse, want_l, 4 * U * want_l, "lse")


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("gap", [18.0, 19.5, 21.0])
@pytest.mark.parametrize("heads,kv_heads,tokens,batch,n,prefix", SHAPES)
def test_f16_keeps_weights_far_below_the_largest(ctx, heads, kv_heads, tokens, batch, n, prefix, gap, d):
    # Every tile of 32 keys begins with a key of score 0 and value 0; the others' weights, e^-gap (2^-26 to 2^-30.3),
    # are all that the result has.
    g = torch.Generator().manual_seed(int(10 * gap) + d)
    k = torch.zeros(2, kv_heads, 512, d)
    k[..., 0] = -gap
    k[:, :, ::32, 0] = 0.0
    v = 500.0 + 500.0 * torch.rand(2, kv_heads, 512, d, generator=g)
    v[:, :, ::32] = 0.0
    v = v.half()
    q = _queries(tokens, heads, d, "f16", 1.0)
    y, lse = _attend(ctx, "f16", "f16", q, k.half().cuda(), v.cuda(), heads, [n] * batch, [[1]] * batch, 512,
                     prefix=prefix, live=min(tokens, batch))
    w = math.exp(-gap)
    vs = torch.cat([v[0, :, :prefix], v[1, :, :n]], 1).double()
    highs = -(-prefix // 32) + -(-n // 32)
    total = highs + w * (prefix + n - highs)
    want = (w * vs.sum(1) / total).repeat_interleave(heads // kv_heads, 0).expand(y.shape)
    # A weight is rounded to 2^-11 of itself, or to half of 2^-24's step where it is below 2^-14: kept 2^7 times as
    # large as it counts, that is 2^-32 of the largest.
    rel = 2.1 * (gap * 1.45 * 2 * U + 4 * U) + (prefix + n) * U + half_step(torch.float16) * 1.01
    bound = want * (rel + 2.0 ** -32 * 1.01 / w + half_step(torch.float16) * 1.01) + smallest(torch.float16)
    assert (bound < 0.6 * want).all()
    within(y, want, bound, "y")


def test_f16_keeps_a_million_small_weights(ctx):
    # one key of score 0 and value 0, and 2^20 - 1 of e^-18, 2^-26, which together are 2^-6 of it
    n, d, page, heads = 1 << 20, 64, 4096, 64
    g = torch.Generator().manual_seed(3)
    k = torch.zeros(2, 1, page, d)
    k[..., 0] = -18.0
    k[0, 0, 0, 0] = 0.0
    v = 1.0 + torch.rand(2, 1, page, d, generator=g)
    v[0, 0, 0] = 0.0
    v = v.half()
    q = _queries(1024, heads, d, "f16", 1.0)
    y, lse = _attend(ctx, "f16", "f16", q, k.half().cuda(), v.cuda(), heads, [n], [[0] + [1] * (n // page - 1)], page,
                     one_range=True, shared=True)
    w = math.exp(-18.0)
    values = v[0, 0].double().sum(0) + (n // page - 1) * v[1, 0].double().sum(0)
    want = (w * values / (1 + w * (n - 1))).expand(y.shape)
    # As above; the products' sum is rounded once for 8 keys at most, the weights' sum at most once a key of a lane
    # and of the four sums that it has, of which one holds the large weight: n / 8 times in two lanes.
    rel = (2.1 * (18 * 1.45 * 2 * U + 4 * U) + n / 8 * U + n / 4 * U + half_step(torch.float16) * 2.02
           + 2.0 ** -32 * 1.01 / w)
    assert rel < 0.05
    within(y, want, want * rel + smallest(torch.float16), "y")
