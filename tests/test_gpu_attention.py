"""Attention over a shared prefix and paged own tokens (vtq_attention_device) against 64 bits."""
import math

import pytest
import torch

import vtq
from serving import TAGS, TYPES, Paged, attention_exact, stream, within

pytestmark = pytest.mark.gpu


def _attend(ctx, p, q, heads, scale, desc=None, tokens=None, y=None, lse=True):
    name = next(k for k, t in TYPES.items() if t == q.dtype)
    desc, tokens = desc or p.desc, q.shape[0] if tokens is None else tokens
    y = torch.full((tokens, heads, p.head_dim), 7.0, dtype=q.dtype, device="cuda") if y is None else y
    l = torch.full((tokens, heads), 7.0, device="cuda")
    need = ctx.attention_workspace(p.cache, desc, TAGS[name], tokens, heads)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")  # NaNs, and a rim that stays
    ctx.attention_device(p.cache, desc, TAGS[name], tokens, heads, q.data_ptr(), q.stride(0), q.stride(1), y.data_ptr(),
                         y.stride(0), y.stride(1), scale, ws.data_ptr(), need, stream(),
                         lse_ptr=l.data_ptr() if lse else None)
    torch.cuda.synchronize()
    assert (ws[need:] == 255).all()
    return y, l


def _case(ctx, q_lens, own_lens, prefix, heads, kv_heads, head_dim, page, name, cache, order="heads", seed=0, big=1.5,
          **more):
    p = Paged(q_lens, own_lens, prefix, kv_heads, head_dim, page, cache, seed=seed, layout=order, **more)
    g = torch.Generator().manual_seed(seed + 1)
    q = (big * torch.randn(p.tokens, heads, head_dim, generator=g)).to(TYPES[name])
    scale = 1.0 / math.sqrt(head_dim)
    y, lse = _attend(ctx, p, q.cuda(), heads, scale)
    want, want_l, by, bl = attention_exact(p, q, heads, float(torch.tensor(scale)))
    within(y, want, by, "y")
    within(lse, want_l, bl, "lse")
    return p, q, y, lse


PAIRS = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]


@pytest.mark.parametrize("name,cache", PAIRS)
@pytest.mark.parametrize("q_lens,own_lens,prefix,heads,kv_heads,head_dim,page", [
    ([1], [1], 0, 1, 1, 8, 8),                                      # one key
    ([1], [1], 1, 4, 1, 64, 16),
    ([1] * 4, [90, 1, 33, 64], 500, 32, 4, 64, 16),
    ([1] * 5, [0, 1, 31, 32, 500], 0, 8, 8, 128, 16),               # one empty row
    ([1, 0, 2, 6, 3], [40, 7, 2, 129, 1000], 100, 24, 8, 96, 32),   # drafts
    ([2, 5], [1, 2], 0, 4, 2, 64, 16),                              # tokens before the first slot: empty rows
    ([2, 5], [1, 2], 35, 4, 2, 64, 16),
    ([70, 33], [70, 300], 65, 7, 1, 80, 64),                        # prompts, group of 7
    ([150], [150], 0, 2, 1, 128, 128),
    ([1] * 40, [3] * 40, 1003, 8, 1, 128, 16),                      # many rows on a prefix
    ([1] * 9, [5] * 9, 4100, 16, 2, 256, 64),
    ([3], [20], 31, 64, 1, 48, 8),                                  # 64 heads on one
    ([1, 1], [2000, 5], 0, 4, 4, 256, 4096),
    ([1], [9000], 0, 8, 8, 64, 16),
    ([0, 0], [5, 0], 10, 4, 2, 64, 16)])                            # nothing to do
def test_attention(ctx, name, cache, q_lens, own_lens, prefix, heads, kv_heads, head_dim, page):
    _case(ctx, q_lens, own_lens, prefix, heads, kv_heads, head_dim, page, name, cache)


@pytest.mark.parametrize("prefix", [0, 1, 7, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513])
def test_prefix_lengths_around_the_tiles(ctx, prefix):
    _case(ctx, [1, 2, 1], [prefix % 67, 2, 33], prefix, 8, 2, 128, 16, "bf16", "bf16", seed=prefix)
    _case(ctx, [20, 13], [20, 40], prefix, 8, 2, 64, 8, "f16", "f16", seed=prefix)


@pytest.mark.parametrize("name,cache,head_dim", [("f32", "f32", 64), ("f32", "bf16", 128), ("bf16", "bf16", 256),
                                                 ("f32", "f32", 256)])
@pytest.mark.parametrize("n", [31, 33, 65, 95, 160, 225, 450, 1000])
def test_parts_of_a_few_tiles(ctx, name, cache, head_dim, n):
    # rows shared by the waves where a tile takes long: parts end at multiples of 32 keys, pages at 8 and 64
    _case(ctx, [1] * 20, [1 + n % 50] * 20, n, 4, 1, head_dim, 8, name, cache, seed=n)
    _case(ctx, [40], [40 + n], n % 37, 2, 1, head_dim, 64, name, cache, seed=n)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("prefix", [128 * n - 3 for n in (2, 3, 5, 9, 16, 17, 25, 33, 50, 63, 64, 65, 80)])
def test_every_number_of_parts(ctx, prefix, head_dim):
    # one row tile of 128 keys a part: the join's groups of lanes see every remainder
    _case(ctx, [1], [5], prefix, 1, 1, head_dim, 16, "bf16", "bf16", seed=prefix)
    _case(ctx, [1], [prefix], 0, 1, 1, head_dim, 16, "f32", "f32", seed=prefix)
    _case(ctx, [1], [prefix], prefix + 1, 1, 1, head_dim, 16, "f16", "f16", seed=prefix)


@pytest.mark.parametrize("name,cache", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")])
def test_slots_before_heads_and_strided_queries(ctx, name, cache):
    p, q, y, lse = _case(ctx, [1, 3], [50, 70], 40, 8, 2, 64, 16, name, cache, order="slots")
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


@pytest.mark.parametrize("name,cache", [("bf16", "bf16"), ("f32", "f16")])
def test_heads_before_pages(ctx, name, cache):
    # heads 2^24 elements and more apart
    _case(ctx, [1, 3], [50, 70], 40, 8, 2, 64, 16, name, cache, order="major", spare_pages=1 << 14)


@pytest.mark.parametrize("name,cache", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("q_lens,prefix", [([1, 2], 0), ([1, 2], 300), ([40, 70], 0), ([40, 70], 300)])
def test_in_place(ctx, name, cache, q_lens, prefix):
    p = Paged(q_lens, [n + 30 for n in q_lens], prefix, 2, 128, 16, cache)
    q = torch.randn(p.tokens, 8, 128, device="cuda").to(TYPES[name])
    want, _ = _attend(ctx, p, q, 8, 0.1)
    y, _ = _attend(ctx, p, q, 8, 0.1, y=q)
    assert y is q and torch.equal(y, want)


def test_rows_behind_the_last_sequence_stay(ctx):
    for prefix, n in ((0, 1), (100, 1), (100, 40), (3000, 1)):
        p = Paged([n, n], [50, 60], prefix, 2, 64, 16, "bf16")
        q = torch.randn(p.tokens + 7, 8, 64, device="cuda").bfloat16()
        y, lse = _attend(ctx, p, q, 8, 0.125)
        assert (y[p.tokens:] == 7.0).all() and (lse[p.tokens:] == 7.0).all()
        y0, lse0 = _attend(ctx, p, q[:p.tokens], 8, 0.125)
        want, wl, by, bl = attention_exact(p, q[:p.tokens].cpu(), 8, 0.125)
        within(y0, want, by, "y")
        within(y[:p.tokens], want, by, "y beside spare rows")


@pytest.mark.parametrize("name,cache", PAIRS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_never_reaches_it(ctx, name, cache, bad):
    # tokens 2, 3 of one sequence hold values that are not finite: tokens 0 and 1 do not see them
    for q_lens, own in (([4], [37]), ([4], [4]), ([40], [90])):
        p, q, y, lse = _case(ctx, q_lens, own, 70, 8, 2, 128, 16, name, cache, seed=5)
        n = q_lens[0]
        first = own[0] - n + 2
        for view in (p.kh, p.vh):
            for place in range(first, own[0]):
                view[int(p.pages[0, place // 16]), :, place % 16, 3:5] = bad
        p.to_device()
        y2, lse2 = _attend(ctx, p, q.cuda(), 8, 1.0 / math.sqrt(128))
        assert torch.equal(y2[:2], y[:2]) and torch.equal(lse2[:2], lse[:2])
        assert not y2[2:, :, 3:5].isfinite().any()


def test_an_infinite_value_gives_infinity_and_a_lowest_score_nothing(ctx):
    p, q, y, lse = _case(ctx, [1], [20], 30, 4, 2, 64, 16, "f32", "f32")
    p.vh[int(p.pages[0, 0]), :, 3, 5] = float("inf")
    p.to_device()
    y2, _ = _attend(ctx, p, q.cuda(), 4, 0.125)
    assert (y2[:, :, 5] == float("inf")).all() and torch.equal(y2[:, :, 6:], y[:, :, 6:])
    # scores of -inf at some keys: as if they were not there
    p, q, y, lse = _case(ctx, [1], [20], 30, 2, 2, 64, 16, "f32", "f32", seed=8)
    q2 = q.abs() + 0.1
    p.kh[int(p.pages[0, 0]), :, 3] = -float("inf")
    p.to_device()
    y3, l3 = _attend(ctx, p, q2.cuda(), 2, 0.125)
    assert y3.isfinite().all() and l3.isfinite().all()


def test_large_scores_and_one_dominant_key(ctx):
    _case(ctx, [1, 2], [300, 5], 200, 8, 2, 128, 16, "f32", "f32", big=60.0, seed=2)
    _case(ctx, [1, 2], [300, 5], 200, 8, 2, 128, 16, "bf16", "bf16", big=60.0, seed=3)


def test_pages_outside_the_cache_count_as_zeros(ctx):
    for name, cache in PAIRS:
        p = Paged([1, 3], [60, 45], 50, 2, 64, 16, cache)
        p.pages[0, 1], p.pages[1, 0], p.prefix_pages[2] = -1, p.n_pages, 2 ** 31 - 1
        p.to_device()
        q = torch.randn(4, 4, 64).to(TYPES[name])
        y, lse = _attend(ctx, p, q.cuda(), 4, 0.125)
        want, wl, by, bl = attention_exact(p, q, 4, 0.125)
        within(y, want, by, "y")
        within(lse, wl, bl, "lse")


def test_lengths_past_the_page_list_are_cut(ctx):
    p = Paged([1, 2], [32, 20], 10, 2, 64, 16, "bf16")
    q = torch.randn(3, 4, 64).bfloat16()
    p.own_lens = [4000, 20]
    p.len[0] = 4000  # the list holds 32
    p.to_device()
    y, lse = _attend(ctx, p, q.cuda(), 4, 0.125)
    want, wl, by, bl = attention_exact(p, q, 4, 0.125)
    within(y, want, by, "y")


@pytest.mark.parametrize("max_q,max_len", [(0, 0), (1, 1), (1, 100000), (500, 0), (7, 64)])
def test_the_hosts_idea_of_the_lengths_only_splits(ctx, max_q, max_len):
    for q_lens, own in (([1, 1, 1], [700, 2, 90]), ([40, 1, 130], [40, 900, 200])):
        p = Paged(q_lens, own, 300, 2, 128, 16, "bf16")
        q = torch.randn(p.tokens, 8, 128).bfloat16()
        y, lse = _attend(ctx, p, q.cuda(), 8, 0.1, desc=p.describe(max_q, max_len))
        want, wl, by, bl = attention_exact(p, q, 8, float(torch.tensor(0.1)))
        within(y, want, by, "y")
        within(lse, wl, bl, "lse")


@pytest.mark.parametrize("name,cache,prefix,q_lens", [("bf16", "bf16", 3000, [1] * 6), ("f32", "f32", 0, [1] * 6),
                                                      ("bf16", "bf16", 700, [50, 1, 1, 20, 1, 1])])
def test_captured_graph_follows_the_lengths(ctx, name, cache, prefix, q_lens):
    p = Paged(q_lens, [900, 400, 60, 100, 7, 1], prefix, 2, 128, 16, cache)
    q = torch.randn(p.tokens, 8, 128, device="cuda").to(TYPES[name])
    ys = [torch.empty_like(q) for _ in range(3)]
    need = ctx.attention_workspace(p.cache, p.desc, TAGS[name], p.tokens, 8)
    wss = [torch.empty(max(need, 256), dtype=torch.uint8, device="cuda") for _ in range(3)]

    def step(i):
        ctx.attention_device(p.cache, p.desc, TAGS[name], p.tokens, 8, q.data_ptr(), q.stride(0), q.stride(1),
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
    p = Paged([1] * 12, [300 + 40 * i for i in range(12)], 2500, 4, 128, 16, "bf16")
    q = torch.randn(12, 16, 128, device="cuda").bfloat16()
    want, wl = _attend(ctx, p, q, 16, 0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):  # two streams at once, a workspace each
        with torch.cuda.stream(streams[i % 2]):
            outs.append(_attend_async(ctx, p, q, 16, 0.1))
    torch.cuda.synchronize()
    for y, l, _ in outs:
        assert torch.equal(y, want) and torch.equal(l, wl)


def _attend_async(ctx, p, q, heads, scale):
    y = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    l = torch.empty(q.shape[:2], device="cuda")
    need = ctx.attention_workspace(p.cache, p.desc, vtq.BF16, q.shape[0], heads)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
    ctx.attention_device(p.cache, p.desc, vtq.BF16, q.shape[0], heads, q.data_ptr(), q.stride(0), q.stride(1),
                         y.data_ptr(), y.stride(0), y.stride(1), scale, ws.data_ptr(), need, stream(),
                         lse_ptr=l.data_ptr())
    return y, l, ws


def test_pages_behind_4_gib(ctx):
    d, page, n_pages = 64, 64, (1 << 31) // (64 * 64) + 100
    kc = torch.empty(n_pages, 1, page, d, dtype=torch.float16, device="cuda")
    vc = torch.empty(n_pages, 1, page, d, dtype=torch.float16, device="cuda")
    last = n_pages - 1
    for c in (kc, vc):
        c[last].normal_()
        c[last - 1].normal_()
    pages = torch.tensor([[last, 0]], dtype=torch.int32, device="cuda")
    prefix = torch.tensor([last - 1], dtype=torch.int32, device="cuda")
    lists = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([60], dtype=torch.int32, device="cuda")
    cache = vtq.KvCache(vtq.F16, kc.data_ptr(), vc.data_ptr(), n_pages, page, 1, d)
    batch = vtq.KvBatch(1, lists[0].data_ptr(), lists[1].data_ptr(), pages.data_ptr(), 2, prefix_len=50,
                        prefix_pages=prefix.data_ptr())
    q = torch.randn(1, 2, d, device="cuda").half()
    y = torch.empty_like(q)
    need = ctx.attention_workspace(cache, batch, vtq.F16, 1, 2)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    ctx.attention_device(cache, batch, vtq.F16, 1, 2, q.data_ptr(), d * 2, d, y.data_ptr(), d * 2, d, 0.125,
                         ws.data_ptr(), need, stream())
    k = torch.cat([kc[last - 1, 0, :50], kc[last, 0, :60]]).double()
    v = torch.cat([vc[last - 1, 0, :50], vc[last, 0, :60]]).double()
    want = torch.softmax(q[0].double() @ k.t() * 0.125, -1) @ v
    assert ((y[0].double() - want).abs() < 4e-3).all()  # fp16 weights and results, values up to 5
