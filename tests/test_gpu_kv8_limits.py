"""Attention over a paged 8-bit cache at the ends of f32's range, and with scales of keys that a row does not see."""
import pytest
import torch

import vtq
from kv8 import Paged8, attention8_exact
from serving import TAGS, TYPES, within
from test_gpu_kv8_attention import _attend

pytestmark = pytest.mark.gpu

LARGEST = 448.0 * 2.0 ** 119  # the greatest value that a cache holds


@pytest.mark.parametrize("head_dim", [16, 64, 128, 256])
@pytest.mark.parametrize("q_lens", [[1] * 5, [70]])
def test_every_finite_f32_query_is_the_sum_of_its_parts(ctx, head_dim, q_lens):
    # One key of 2^-117 in element 0 and zeros: a row that sees it alone has the score q[0] * 2^-117, which is its lse (scale
    # 1), exactly; the other elements, as large, meet zeros.
    g = torch.Generator().manual_seed(head_dim)
    p = Paged8(q_lens, q_lens, 0, 1, head_dim, 16, fill=False)
    p.kc.zero_(), p.vc.zero_()
    p.view(p.kc)[..., 0] = 0x38
    p.ks.fill_(127 - 117), p.vs.fill_(127)
    p.to_device()
    top = torch.finfo(torch.float32).max
    q = torch.empty(p.tokens, 8, head_dim).uniform_(0.98, 1.0, generator=g) * top
    q *= torch.randint(0, 2, q.shape, generator=g) * 2.0 - 1.0
    q[:, 1] = top
    q[:, 2] = -top
    q[:, 3, 0] = torch.randn(p.tokens, generator=g) * 1e30
    q[:, 4, 0] = 3.3961775e38  # the first f32 number that rounds to no finite bf16
    _, lse = _attend(ctx, p, q.cuda(), 8, 1.0)
    # (every key is alike: a row that sees n has ln n more, below half a step of all but the smallest scores)
    want = q[..., 0] * 2.0 ** -117
    assert want.isfinite().all()
    if q_lens[0] == 1:
        assert torch.equal(lse.cpu(), want)
    else:
        assert ((lse.cpu() - want).abs() <= 5.0 + want.abs() * 2.0 ** -23).all()


def test_infinite_f32_queries_stay_infinite(ctx):
    # beside the split of the largest finite ones: an infinity times a positive key is an infinite score, times zero none
    p = Paged8([1, 1], [1, 1], 0, 1, 16, 16, fill=False)
    p.kc.zero_(), p.vc.fill_(0x38)
    p.view(p.kc)[..., 0] = 0x38
    p.ks.fill_(127), p.vs.fill_(127)
    p.to_device()
    q = torch.zeros(2, 2, 16)
    q[0, 0, 0] = float("inf")
    q[0, 1, 3] = float("inf")
    q[1, 0, 0] = 1.0
    y, lse = _attend(ctx, p, q.cuda(), 2, 1.0)
    assert y[0].isnan().all() and y[1].eq(1.0).all() and lse[1].tolist() == [1.0, 0.0]


def _near(y, name, value):
    # sums of weights in f32, their rounded parts, the quotient and y: 2^-7 of bf16, 2^-13 of f32 at most
    return (y.double() / value - 1).abs().max() <= (2 ** -7 if name == "bf16" else 2 ** -13)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("exponent", [0, 16, 20, 60, 95])
@pytest.mark.parametrize("q_lens,own,prefix", [([1, 1], [20, 300], 0), ([1, 3], [700, 40], 900), ([40], [70], 40),
                                               ([1], [33], 2000)])
def test_sums_of_the_largest_values_under_large_scores(ctx, name, exponent, q_lens, own, prefix):
    # every key alike, with scores from 3e4 to 1e33, and every value the largest: their mean is one, their sum is none in f32
    for head_dim in (64, 128, 192):
        p = Paged8(q_lens, own, prefix, 1, head_dim, 16, fill=False)
        p.kc.fill_(0x7E), p.vc.fill_(0x7E)
        p.ks.fill_(127 + exponent), p.vs.fill_(246)
        p.to_device()
        q = torch.ones(p.tokens, 4, head_dim, dtype=TYPES[name])
        y, _ = _attend(ctx, p, q.cuda(), 4, 1.0)
        assert _near(y, name, LARGEST), (head_dim, y.flatten()[0])


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("byte", [222, 246])
def test_sums_of_many_large_values(ctx, name, byte):
    # 2^17 keys of one score behind 64 of a score 7.5 powers of two below it, so that a maximum of the first ones gives the
    # others weights above 1; a sequence a workgroup, all reading the same pages
    batch, page, heads, head_dim, keys = 512, 4096, 64, 64, 1 << 17
    kc, vc = (torch.zeros(2, 1, page, head_dim, dtype=torch.uint8, device="cuda") for _ in range(2))
    vc.fill_(0x7E)
    kc[..., 0] = 0x38              # 1
    kc[0, 0, :64] = 0              # 0
    ks, vs = (torch.full((2, 1, page // 16), b, dtype=torch.uint8, device="cuda") for b in (127, byte))
    pages = torch.ones(batch, keys // page, dtype=torch.int32, device="cuda")
    pages[:, 0] = 0
    q_start = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    lens = torch.full((batch,), keys, dtype=torch.int32, device="cuda")
    cache = vtq.Kv8Cache(kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), 2, page, 1, head_dim)
    desc = vtq.KvBatch(batch, q_start.data_ptr(), lens.data_ptr(), pages.data_ptr(), keys // page)
    q = torch.zeros(batch, heads, head_dim, device="cuda", dtype=TYPES[name])
    q[..., 0] = 5.1875  # times log2 e: 7.48
    y = torch.zeros_like(q)
    need = ctx.kv8_attention_workspace(cache, desc, TAGS[name], batch, heads)
    ws = torch.full((max(need, 256),), 255, dtype=torch.uint8, device="cuda")
    at = (heads * head_dim, head_dim)
    ctx.kv8_attention_device(cache, desc, TAGS[name], batch, heads, q.data_ptr(), *at, y.data_ptr(), *at, 1.0, ws.data_ptr(),
                             need, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    value = 448.0 * 2.0 ** (byte - 127)
    # a sum of 2^17 equal weights one after another in f32 may be off by 2^17 half steps, 2^-7, as may that of the values
    assert (y.double() / value - 1).abs().max() <= 2 ** -6 + 2 ** -7


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 2), (64, 2)])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_scales_of_values_that_a_row_does_not_see(ctx, name, heads, kv_heads, head_dim):
    # tokens 0 to 11 see the first two blocks alone: whatever scale the third one has, they are the same
    p = Paged8([20], [40], 0, kv_heads, head_dim, 16, seed=3)
    q = torch.randn(20, heads, head_dim, generator=torch.Generator().manual_seed(1)).to(TYPES[name])
    y, lse = _attend(ctx, p, q.cuda(), heads, 0.125)
    for byte in (0, 200, 222, 223, 246, 255):
        p.scale_view(p.vs)[int(p.pages[0, 2])] = byte
        p.to_device()
        y2, lse2 = _attend(ctx, p, q.cuda(), heads, 0.125)
        assert torch.equal(y2[:12], y[:12]), byte
        assert torch.equal(lse2, lse), byte


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,own,prefix,heads,kv_heads,head_dim", [
    ([1, 3], [700, 40], 900, 8, 2, 64), ([1], [3000], 0, 4, 1, 128), ([40, 9], [90, 300], 500, 8, 2, 256),
    ([1] * 40, [30] * 40, 2000, 16, 2, 128), ([130], [130], 33, 4, 2, 64)])
def test_zeros_under_any_scale_are_zeros(ctx, name, q_lens, own, prefix, heads, kv_heads, head_dim):
    # blocks of zeros here and there, once under the least scales and once under the greatest: the same rows, bit for bit
    p = Paged8(q_lens, own, prefix, kv_heads, head_dim, 32, seed=6)
    g = torch.Generator().manual_seed(2)
    zeros = torch.rand(p.vs.shape, generator=g) < 0.1
    p.vc[zeros.repeat_interleave(16, -1)] = 0
    q = torch.randn(p.tokens, heads, head_dim, generator=g).to(TYPES[name]).cuda()
    seen = []
    for byte in (10, 127, 246):
        p.vs[zeros] = byte
        p.to_device()
        seen.append(_attend(ctx, p, q, heads, 0.1))
    for y, lse in seen[1:]:
        assert y.isfinite().all() and torch.equal(y, seen[0][0]) and torch.equal(lse, seen[0][1])


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_large_blocks_among_small_ones(ctx, name):
    # some sequences' blocks, and some ranges of the prefix, up to 2^30 below f32's end, the others as they come
    for q_lens, own, prefix, head_dim in (([1, 3, 1], [700, 40, 5], 900, 64), ([40, 9], [90, 300], 2500, 128),
                                          ([1, 1], [33, 4000], 0, 192)):
        p = Paged8(q_lens, own, prefix, 2, head_dim, 16, seed=8)
        g = torch.Generator().manual_seed(9)
        high = torch.rand(p.vs.shape, generator=g) < 0.2
        p.vs[high] = torch.randint(180, 215, p.vs.shape, generator=g, dtype=torch.uint8)[high]
        p.refresh()
        p.to_device()
        q = torch.randn(p.tokens, 8, head_dim, generator=g).to(TYPES[name])
        y, lse = _attend(ctx, p, q.cuda(), 8, 0.125)
        want, want_l, by, bl = attention8_exact(p, q, 8, 0.125)
        within(y, want, by, "y")
        within(lse, want_l, bl, "lse")
