"""Attention over a paged 8-bit cache (vtq_kv8_attention_device) against 64 bits."""
import math

import pytest
import torch

import vtq
from kv8 import Paged8, attention8_exact
from serving import TAGS, TYPES, stream, within
from vtq import probe

pytestmark = pytest.mark.gpu

NAMES = ["f32", "f16", "bf16"]


def _attend(ctx, p, q, heads, scale, desc=None, y=None, lse=True, wait=True):
    name = next(k for k, t in TYPES.items() if t == q.dtype)
    desc, tokens = desc or p.desc, q.shape[0]
    y = torch.full((tokens, heads, p.head_dim), 7.0, dtype=q.dtype, device="cuda") if y is None else y
    l = torch.full((tokens, heads), 7.0, device="cuda")
    need = ctx.kv8_attention_workspace(p.cache, desc, TAGS[name], tokens, heads)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")  # NaNs, and a rim that stays
    ctx.kv8_attention_device(p.cache, desc, TAGS[name], tokens, heads, q.data_ptr(), q.stride(0), q.stride(1),
                             y.data_ptr(), y.stride(0), y.stride(1), scale, ws.data_ptr(), need, stream(),
                             lse_ptr=l.data_ptr() if lse else None)
    if wait:
        torch.cuda.synchronize()
        assert (ws[need:] == 255).all()
        return y, l
    return y, l, ws


def _case(ctx, q_lens, own_lens, prefix, heads, kv_heads, head_dim, page, name, block=16, order="heads", seed=0, big=1.5,
          **more):
    p = Paged8(q_lens, own_lens, prefix, kv_heads, head_dim, page, block, seed=seed, layout=order, **more)
    g = torch.Generator().manual_seed(seed + 1)
    q = (big * torch.randn(p.tokens, heads, head_dim, generator=g)).to(TYPES[name])
    scale = 1.0 / math.sqrt(head_dim)
    y, lse = _attend(ctx, p, q.cuda(), heads, scale)
    want, want_l, by, bl = attention8_exact(p, q, heads, float(torch.tensor(scale)))
    within(y, want, by, "y")
    within(lse, want_l, bl, "lse")
    return p, q, y, lse


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("q_lens,own_lens,prefix,heads,kv_heads,head_dim,page,block", [
    ([1], [1], 0, 1, 1, 16, 16, 16),                                    # one key
    ([1], [1], 1, 4, 1, 64, 16, 16),
    ([1] * 4, [90, 1, 33, 64], 500, 32, 4, 64, 16, 16),
    ([1] * 5, [0, 1, 31, 32, 500], 0, 8, 8, 128, 16, 16),               # one empty row
    ([1, 0, 2, 6, 3], [40, 7, 2, 129, 1000], 100, 24, 8, 96, 32, 16),   # drafts
    ([2, 5], [1, 2], 0, 4, 2, 64, 16, 16),                              # tokens before the first slot: empty rows
    ([2, 5], [1, 2], 35, 4, 2, 64, 16, 16),
    ([70, 33], [70, 300], 65, 7, 1, 80, 64, 32),                        # prompts, group of 7
    ([150], [150], 0, 2, 1, 128, 128, 128),
    ([1] * 40, [3] * 40, 1003, 8, 1, 128, 16, 16),                      # many rows on a prefix
    ([1] * 9, [5] * 9, 4100, 16, 2, 256, 64, 64),
    ([3], [20], 31, 64, 1, 48, 16, 16),                                 # 64 heads on one
    ([1, 1], [2000, 5], 0, 4, 4, 256, 4096, 256),
    ([1], [9000], 0, 8, 8, 64, 16, 16),
    ([90], [5000], 0, 2, 1, 112, 32, 16),                               # more than 1024 keys to a workgroup
    ([0, 0], [5, 0], 10, 4, 2, 64, 16, 16)])                            # nothing to do
def test_attention(ctx, name, q_lens, own_lens, prefix, heads, kv_heads, head_dim, page, block):
    _case(ctx, q_lens, own_lens, prefix, heads, kv_heads, head_dim, page, name, block)


@pytest.mark.parametrize("prefix", [0, 1, 7, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513])
def test_prefix_lengths_around_the_tiles(ctx, prefix):
    _case(ctx, [1, 2, 1], [prefix % 67, 2, 33], prefix, 8, 2, 128, 16, "bf16", seed=prefix)
    _case(ctx, [20, 13], [20, 40], prefix, 8, 2, 64, 32, "f16", seed=prefix)
    _case(ctx, [20, 13], [20, 40], prefix, 4, 1, 256, 32, "bf16", seed=prefix)


@pytest.mark.parametrize("name,head_dim", [("f32", 64), ("f32", 128), ("bf16", 256), ("f32", 256)])
@pytest.mark.parametrize("n", [31, 33, 65, 95, 160, 225, 450, 1000])
def test_parts_of_a_few_tiles(ctx, name, head_dim, n):
    _case(ctx, [1] * 20, [1 + n % 50] * 20, n, 4, 1, head_dim, 16, name, seed=n)
    _case(ctx, [40], [40 + n], n % 37, 2, 1, head_dim, 64, name, seed=n)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("prefix", [128 * n - 3 for n in (2, 3, 5, 9, 17, 33, 64, 80)])
def test_many_parts(ctx, prefix, head_dim):
    _case(ctx, [1], [5], prefix, 1, 1, head_dim, 16, "bf16", seed=prefix)
    _case(ctx, [1], [prefix], 0, 1, 1, head_dim, 16, "f32", seed=prefix)
    _case(ctx, [1], [prefix], prefix + 1, 1, 1, head_dim, 16, "f16", seed=prefix)


@pytest.mark.parametrize("name", NAMES)
def test_slots_before_heads_and_strided_queries(ctx, name):
    p, q, y, lse = _case(ctx, [1, 3], [50, 70], 40, 8, 2, 64, 16, name, order="slots")
    # queries inside packed rows, results into others, no lse
    packed = torch.full((p.tokens, 12, 64), 3.0, dtype=q.dtype, device="cuda")
    packed[:, 1:9] = q.cuda()
    out = torch.full((p.tokens, 10, 64), 5.0, dtype=q.dtype, device="cuda")
    _attend(ctx, p, packed[:, 1:9], 8, 0.125, y=out[:, 1:9], lse=False)
    assert torch.equal(out[:, 1:9], y) and (out[:, 0] == 5.0).all() and (out[:, 9] == 5.0).all()
    # heads before tokens
    swapped = q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    y2, _ = _attend(ctx, p, swapped, 8, 0.125)
    assert torch.equal(y2, y)


@pytest.mark.parametrize("name", NAMES)
def test_heads_before_pages(ctx, name):
    _case(ctx, [1, 3], [50, 70], 40, 8, 2, 64, 32, name, order="major", spare_pages=1 << 12)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("q_lens,prefix", [([1, 2], 0), ([1, 2], 300), ([40, 70], 0), ([40, 70], 300)])
def test_in_place(ctx, name, q_lens, prefix):
    p = Paged8(q_lens, [n + 30 for n in q_lens], prefix, 2, 128, 16)
    q = torch.randn(p.tokens, 8, 128, device="cuda").to(TYPES[name])
    want, _ = _attend(ctx, p, q, 8, 0.1)
    y, _ = _attend(ctx, p, q, 8, 0.1, y=q)
    assert y is q and torch.equal(y, want)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("q_lens,own", [([1] * 64, 20), ([200, 70], 300), ([3] * 300, 40)])
def test_in_place_of_long_heads(ctx, name, q_lens, own):
    # two workgroups read a row of more than 128 elements, and each writes half of it
    p = Paged8(q_lens, [max(own, n) for n in q_lens], 0, 2, 256, 16)
    q = torch.randn(p.tokens, 8, 256, device="cuda").to(TYPES[name])
    want, _ = _attend(ctx, p, q, 8, 0.1)
    y, _ = _attend(ctx, p, q, 8, 0.1, y=q)
    assert y is q and torch.equal(y, want)


def test_rows_behind_the_last_sequence_stay(ctx):
    for prefix, n in ((0, 1), (100, 1), (100, 40), (3000, 1)):
        p = Paged8([n, n], [50, 60], prefix, 2, 64, 16)
        q = torch.randn(p.tokens + 7, 8, 64, device="cuda").bfloat16()
        y, lse = _attend(ctx, p, q, 8, 0.125)
        assert (y[p.tokens:] == 7.0).all() and (lse[p.tokens:] == 7.0).all()
        want, wl, by, bl = attention8_exact(p, q[:p.tokens].cpu(), 8, 0.125)
        within(y[:p.tokens], want, by, "y beside spare rows")


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("head_dim", [64, 128, 144])
@pytest.mark.parametrize("prefix", [0, 70])
def test_the_longest_sequence_is_only_a_hint(ctx, name, head_dim, prefix):
    # which rows are multiplied 16, 32 or 128 at a time is chosen by it
    p = Paged8([1, 70, 5, 33], [30, 90, 5, 400], prefix, 2, head_dim, 16, seed=4)
    q = torch.randn(p.tokens, 8, head_dim, generator=torch.Generator().manual_seed(6)).to(TYPES[name])
    want, want_l, by, bl = attention8_exact(p, q, 8, 0.125)
    for max_q, max_len in ((0, 0), (1, 0), (4, 1), (5, 400), (70, 100000), (100000, 17)):
        y, lse = _attend(ctx, p, q.cuda(), 8, 0.125, desc=p.describe(max_q=max_q, max_len=max_len))
        within(y, want, by, f"y by {max_q}, {max_len}")
        within(lse, want_l, bl, "lse")


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("head_dim,prefix", [(64, 1), (64, 70), (128, 33), (128, 200), (256, 64)])
def test_prompts_behind_a_short_prefix(ctx, name, head_dim, prefix):
    # prompts that fill the chip take the prefix's keys in their own workgroups; among them tokens without a slot, which
    # see the prefix alone, and a sequence without tokens
    q_lens = [33] * 30 + [1, 0, 70, 40, 5] + [20] * 31
    own = [40] * 30 + [1, 7, 90, 30, 0] + [25] * 31
    p = Paged8(q_lens, own, prefix, 4, head_dim, 16, seed=prefix)
    assert probe.attention_plan(p.cache, p.desc, TAGS[name], p.tokens, 8)["prefix_splits"] == 0
    q = torch.randn(p.tokens, 8, head_dim, generator=torch.Generator().manual_seed(8)).to(TYPES[name])
    y, lse = _attend(ctx, p, q.cuda(), 8, 0.2)
    want, want_l, by, bl = attention8_exact(p, q, 8, 0.2)
    within(y, want, by, "y")
    within(lse, want_l, bl, "lse")
    z = q.cuda()
    _attend(ctx, p, z, 8, 0.2, y=z)
    assert torch.equal(z, y)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (16, 1), (17, 1), (14, 2)])
def test_rows_of_a_group_around_16(ctx, name, heads, kv_heads):
    for head_dim in (64, 128, 256):
        _case(ctx, [1, 1, 1], [1, 333, 2000], 45, heads, kv_heads, head_dim, 16, name, seed=heads)
        _case(ctx, [3, 2], [40, 2], 0, heads, kv_heads, head_dim, 32, name, block=32, seed=heads)
        # the last key of each row no number, which the row before does not see
        p, q, y, lse = _case(ctx, [3], [50], 0, heads, kv_heads, head_dim, 16, name, seed=heads + 1)
        p.view(p.vc)[int(p.pages[0, 49 // 16]), :, 49 % 16, ::7] = 0x7F
        p.refresh()
        p.to_device()
        y2, _ = _attend(ctx, p, q.cuda(), heads, 1.0 / math.sqrt(head_dim))
        assert torch.equal(y2[:2], y[:2])
        assert y2[2, :, ::7].isnan().all()
        rest = torch.arange(head_dim) % 7 != 0
        assert torch.equal(y2[2][:, rest], y[2][:, rest])


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_what_a_row_does_not_see_never_reaches_it(ctx, name, head_dim):
    # tokens from 2 on of one sequence hold NaN in elements 3 and 4: tokens 0 and 1 do not see them
    for q_lens, own in (([4], [37]), ([4], [4]), ([40], [90])):
        p, q, y, lse = _case(ctx, q_lens, own, 70, 8, 2, head_dim, 16, name, seed=5)
        first = own[0] - q_lens[0] + 2
        for codes in (p.kc, p.vc):
            for place in range(first, own[0]):
                p.view(codes)[int(p.pages[0, place // 16]), :, place % 16, 3:5] = 0xFF
        p.refresh()
        p.to_device()
        y2, lse2 = _attend(ctx, p, q.cuda(), 8, 1.0 / math.sqrt(head_dim))
        assert torch.equal(y2[:2], y[:2]) and torch.equal(lse2[:2], lse[:2])
        assert y2[2:].isnan().all()  # a key that is no number leaves no row that sees it a number
        # in the values alone: those elements, and no others
        p2 = Paged8(q_lens, own, 70, 2, head_dim, 16, seed=5)
        for place in range(first, own[0]):
            p2.view(p2.vc)[int(p2.pages[0, place // 16]), :, place % 16, 3:5] = 0x7F
        p2.to_device()
        y3, lse3 = _attend(ctx, p2, q.cuda(), 8, 1.0 / math.sqrt(head_dim))
        assert torch.equal(y3[:2], y[:2]) and torch.equal(lse3, lse)
        assert y3[2:, :, 3:5].isnan().all()
        assert torch.equal(y3[..., 5:], y[..., 5:]) and torch.equal(y3[..., :3], y[..., :3])


@pytest.mark.parametrize("name", NAMES)
def test_scales_far_apart(ctx, name):
    # blocks 2^60 apart: what a small one adds to a large one is lost in the sum of magnitudes, and no more
    for seed in range(3):
        p = Paged8([1, 3], [100, 70], 90, 2, 64, 16, seed=seed)
        g = torch.Generator().manual_seed(seed)
        p.vs += torch.randint(-60, 61, p.vs.shape, generator=g).to(torch.int8).view(torch.uint8)
        p.ks += torch.randint(-6, 3, p.ks.shape, generator=g).to(torch.int8).view(torch.uint8)
        p.refresh()
        p.to_device()
        q = torch.randn(4, 4, 64, generator=g).to(TYPES[name])
        y, lse = _attend(ctx, p, q.cuda(), 4, 0.125)
        want, wl, by, bl = attention8_exact(p, q, 4, 0.125)
        if name != "f16":  # most results are past its range
            within(y, want, by, "y")
        within(lse, wl, bl, "lse")


def test_bytes_of_scales_outside_their_range(ctx):
    p = Paged8([1, 1], [20, 20], 0, 1, 16, 16)
    for i, byte in enumerate((0, 9, 5, 3)):  # all as 10
        p.vs[int(p.pages[i // 2, i % 2])] = byte
    p.refresh()
    p.to_device()
    q = torch.randn(2, 1, 16)
    y, _ = _attend(ctx, p, q.cuda(), 1, 0.25)
    want, _, by, _ = attention8_exact(p, q, 1, 0.25)
    assert (want.abs() > 0).all() and (y != 0).any()
    within(y, want, by, "y")
    for i, byte in enumerate((255, 247, 254, 250)):  # as 246
        p.vs[int(p.pages[i // 2, i % 2])] = byte
    p.refresh()
    p.to_device()
    y2, _ = _attend(ctx, p, q.cuda(), 1, 0.25)
    want, _, by, _ = attention8_exact(p, q, 1, 0.25)
    within(y2, want, by, "y of the largest scale")
    assert y2.isfinite().all()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_sums_of_the_largest_values(ctx, name):
    # every value 448 x 2^119: their weighted mean is one too, their sum is none in f32
    for q_lens, own, prefix in (([1, 1], [20, 300], 0), ([1, 3], [700, 40], 900), ([40], [70], 40), ([1], [33], 2000)):
        for head_dim in (64, 128, 192):
            p = Paged8(q_lens, own, prefix, 1, head_dim, 16)
            p.vc.fill_(0x7E)
            p.vs.fill_(246)
            p.to_device()
            q = torch.randn(p.tokens, 4, head_dim, generator=torch.Generator().manual_seed(3)).to(TYPES[name])
            y, _ = _attend(ctx, p, q.cuda(), 4, head_dim**-0.5)
            # sums of weights in f32, their rounded parts, the quotient and y: 2^-7 of bf16, 2^-13 of f32 at most
            assert (y.double() / (448 * 2.0**119) - 1).abs().max() <= (2**-7 if name == "bf16" else 2**-13)


def test_large_scores_and_one_dominant_key(ctx):
    for name in NAMES:
        _case(ctx, [1, 2], [300, 5], 200, 8, 2, 128, 16, name, big=60.0, seed=2)


def test_scores_in_the_millions(ctx):
    # keys so loud that a row's best score alone counts, and scores' differences before the scale
    for name in NAMES:
        _case(ctx, [1, 2], [60, 33], 40, 4, 2, 64, 16, name, big=3000.0, loud=3000.0, seed=4)


def test_infinite_queries(ctx):
    # an infinite element gives its row no number, as q . k then is none or infinite; the others stay
    p = Paged8([1, 1], [40, 40], 0, 1, 64, 16)
    for name in NAMES:
        q = torch.randn(2, 4, 64).to(TYPES[name])
        y, _ = _attend(ctx, p, q.cuda(), 4, 0.125)
        q2 = q.clone()
        q2[0, 1, 7] = float("inf")
        q2[1, 2, 9] = float("nan")
        y2, _ = _attend(ctx, p, q2.cuda(), 4, 0.125)
        keep = torch.ones(2, 4, dtype=torch.bool)
        keep[0, 1] = keep[1, 2] = False
        assert torch.equal(y2.cpu()[keep], y.cpu()[keep]) and y2[1, 2].isnan().all()


def test_pages_outside_the_cache_count_as_zeros(ctx):
    for name in NAMES:
        p = Paged8([1, 3], [60, 45], 50, 2, 64, 16)
        p.pages[0, 1], p.pages[1, 0], p.prefix_pages[2] = -1, p.n_pages, 2 ** 31 - 1
        p.to_device()
        q = torch.randn(4, 4, 64).to(TYPES[name])
        y, lse = _attend(ctx, p, q.cuda(), 4, 0.125)
        want, wl, by, bl = attention8_exact(p, q, 4, 0.125)
        within(y, want, by, "y")
        within(lse, wl, bl, "lse")


def test_lengths_past_the_page_list_are_cut(ctx):
    p = Paged8([1, 2], [32, 20], 10, 2, 64, 16)
    q = torch.randn(3, 4, 64).bfloat16()
    p.own_lens = [4000, 20]
    p.len[0] = 4000  # the list holds 32
    p.to_device()
    y, lse = _attend(ctx, p, q.cuda(), 4, 0.125)
    want, wl, by, bl = attention8_exact(p, q, 4, 0.125)
    within(y, want, by, "y")


@pytest.mark.parametrize("max_q,max_len", [(0, 0), (1, 1), (1, 100000), (500, 0), (7, 64)])
def test_the_hosts_idea_of_the_lengths_only_splits(ctx, max_q, max_len):
    for q_lens, own in (([1, 1, 1], [700, 2, 90]), ([40, 1, 130], [40, 900, 200])):
        p = Paged8(q_lens, own, 300, 2, 128, 16)
        q = torch.randn(p.tokens, 8, 128).bfloat16()
        y, lse = _attend(ctx, p, q.cuda(), 8, 0.1, desc=p.describe(max_q, max_len))
        want, wl, by, bl = attention8_exact(p, q, 8, float(torch.tensor(0.1)))
        within(y, want, by, "y")
        within(lse, wl, bl, "lse")


@pytest.mark.parametrize("name,prefix,q_lens", [("bf16", 3000, [1] * 6), ("f32", 0, [1] * 6),
                                                ("bf16", 700, [50, 1, 1, 20, 1, 1])])
def test_captured_graph_follows_the_lengths(ctx, name, prefix, q_lens):
    p = Paged8(q_lens, [900, 400, 60, 100, 7, 1], prefix, 2, 128, 16)
    q = torch.randn(p.tokens, 8, 128, device="cuda").to(TYPES[name])
    ys = [torch.empty_like(q) for _ in range(3)]
    need = ctx.kv8_attention_workspace(p.cache, p.desc, TAGS[name], p.tokens, 8)
    wss = [torch.empty(max(need, 256), dtype=torch.uint8, device="cuda") for _ in range(3)]

    def step(i):
        ctx.kv8_attention_device(p.cache, p.desc, TAGS[name], p.tokens, 8, q.data_ptr(), q.stride(0), q.stride(1),
                                 ys[i].data_ptr(), q.stride(0), q.stride(1), 0.09, wss[i].data_ptr(), need, stream())

    step(0)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            step(i + 1)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device="cuda"))
        if i:
            p.dlists[1].copy_(torch.tensor([900 - 200 * i, 400 - i, 60, 100 - i, 7, 1], dtype=torch.int32))
        for y in ys:
            y.fill_(float("nan"))
        for ws in wss:
            ws.fill_(255)
        for graph in graphs:
            graph.replay()
        step(0)
        torch.cuda.synchronize()
        assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2]) and ys[0].isfinite().all()


def test_the_same_call_gives_the_same_bits_on_any_stream(ctx):
    p = Paged8([1] * 12, [300 + 40 * i for i in range(12)], 2500, 4, 128, 16)
    q = torch.randn(12, 16, 128, device="cuda").bfloat16()
    want, wl = _attend(ctx, p, q, 16, 0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):  # two streams at once, a workspace each
        with torch.cuda.stream(streams[i % 2]):
            outs.append(_attend(ctx, p, q, 16, 0.1, wait=False))
    torch.cuda.synchronize()
    for y, l, _ in outs:
        assert torch.equal(y, want) and torch.equal(l, wl)


def test_pages_behind_4_gib(ctx):
    d, page, n_pages = 64, 64, (1 << 32) // (64 * 64) + 100
    kc, vc = (torch.empty(n_pages, 1, page, d, dtype=torch.uint8, device="cuda") for _ in range(2))
    scales = torch.full((2, n_pages, 1, page // 16), 127, dtype=torch.uint8, device="cuda")
    last = n_pages - 1
    for c in (kc, vc):
        for i in (last, last - 1):
            c[i] = torch.randn(1, page, d, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
    scales[:, last] = 126
    pages = torch.tensor([[last, 0]], dtype=torch.int32, device="cuda")
    prefix = torch.tensor([last - 1], dtype=torch.int32, device="cuda")
    lists = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([60], dtype=torch.int32, device="cuda")
    cache = vtq.Kv8Cache(kc.data_ptr(), vc.data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), n_pages, page, 1, d)
    batch = vtq.KvBatch(1, lists[0].data_ptr(), lists[1].data_ptr(), pages.data_ptr(), 2, prefix_len=50,
                        prefix_pages=prefix.data_ptr())
    q = torch.randn(1, 2, d, device="cuda").half()
    y = torch.empty_like(q)
    need = ctx.kv8_attention_workspace(cache, batch, vtq.F16, 1, 2)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    ctx.kv8_attention_device(cache, batch, vtq.F16, 1, 2, q.data_ptr(), d * 2, d, y.data_ptr(), d * 2, d, 0.125,
                             ws.data_ptr(), need, stream())
    real = [torch.cat([c[last - 1, 0, :50].view(torch.float8_e4m3fn).double(),
                       c[last, 0, :60].view(torch.float8_e4m3fn).double() * 0.5]) for c in (kc, vc)]
    want = torch.softmax(q[0].double() @ real[0].t() * 0.125, -1) @ real[1]
    # f16 results up to 5: 2^-11 of that, and weights to 2^-16
    assert ((y[0].double() - want).abs() < 3e-3).all()
