"""Appending to a paged 8-bit cache (vtq_kv8_append_device) against its definition in 64 bits."""
import pytest
import torch

import vtq
from kv8 import Paged8, append8_exact, same_codes
from serving import TAGS, TYPES, frequencies, rotate_exact, rotation_bound, smallest, stream, within

pytestmark = pytest.mark.gpu

HALF, INTER = vtq.ROPE_HALF, vtq.ROPE_INTERLEAVED


def _append(ctx, p, rope, name, k, v, q=None, out=None, desc=None):
    args = {}
    if q is not None:
        args = dict(heads=q.shape[1], q_ptr=q.data_ptr(), q_token_stride=q.stride(0), q_head_stride=q.stride(1),
                    q_out_ptr=out.data_ptr(), q_out_token_stride=out.stride(0), q_out_head_stride=out.stride(1))
    ctx.kv8_append_device(p.cache, desc or p.desc, rope, TAGS[name], k.shape[0], k.data_ptr(), k.stride(0), k.stride(1),
                          v.data_ptr(), v.stride(0), v.stride(1), stream(), **args)
    torch.cuda.synchronize()


def _check(p, packed, heads, rot, layout, name):
    """The cache on the device after the tokens of `packed` went into the state that p holds."""
    hk = p.kv_heads
    pos = torch.tensor([p.prefix + place for _, place in p.places()], dtype=torch.int64)
    x = packed[:p.tokens, heads:heads + hk]
    if rot:
        freq, m = frequencies(rot)
        want, size, _ = rotate_exact(x, pos, freq, m, layout)
        off = 5 * 2.0 ** -24 * size + smallest(torch.float32)
    else:
        want, off = x.double(), torch.zeros_like(x, dtype=torch.float64)
    append8_exact(p, "k", want, off)
    v = packed[:p.tokens, heads + hk:].double()
    append8_exact(p, "v", v, torch.zeros_like(v))


def _case(ctx, q_lens, own_lens, prefix, heads, kv_heads, head_dim, rot, layout, page, block, name, order="heads", seed=0,
          spare_tokens=0, change=None, loud=1.0):
    p = Paged8(q_lens, own_lens, prefix, kv_heads, head_dim, page, block, seed=seed, layout=order)
    if change:
        change(p)
        p.refresh()
        p.to_device()
    g = torch.Generator().manual_seed(seed + 1)
    tokens = p.tokens + spare_tokens
    packed = torch.randn(tokens, heads + 2 * kv_heads, head_dim, generator=g)
    packed = (packed * torch.exp2(loud * torch.randn(tokens, heads + 2 * kv_heads, 1, generator=g))).to(TYPES[name])
    dev = packed.cuda()
    q, k, v = dev.split([heads, kv_heads, kv_heads], 1)
    out = torch.full((tokens, heads, head_dim), 7.0, dtype=q.dtype, device="cuda")
    _append(ctx, p, vtq.Rope(rot, layout) if rot else None, name, k, v, q if heads else None, out)
    _check(p, packed, heads, rot, layout, name)
    if heads:
        pos = torch.tensor([prefix + place for _, place in p.places()], dtype=torch.int64)
        freq, m = frequencies(rot) if rot else (torch.zeros(0, dtype=torch.float64), 1.0)
        want, size, _ = rotate_exact(packed[:p.tokens, :heads], pos, freq, m, layout)
        within(out[:p.tokens], want, rotation_bound(want, size, q.dtype), "queries")
        assert (out[p.tokens:] == 7.0).all()
    return p, dev


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,own_lens,prefix,heads,kv_heads,head_dim,rot,layout,page,block", [
    ([1], [1], 0, 1, 1, 16, 16, HALF, 16, 16),
    ([1] * 5, [1, 16, 17, 300, 64], 2000, 32, 8, 128, 128, HALF, 16, 16),
    ([3, 0, 7, 1, 0], [3, 9, 40, 1, 0], 77, 4, 4, 64, 32, INTER, 32, 16),
    ([40, 17], [40, 100], 0, 7, 1, 80, 80, HALF, 64, 32),
    ([130], [130], 5, 6, 2, 96, 24, INTER, 16, 16),
    ([100, 33], [105, 70], 5, 6, 2, 64, 12, HALF, 128, 128),     # N = 1; blocks of 128 tokens
    ([2, 2], [5, 4097], 1, 8, 8, 256, 64, HALF, 4096, 4096),
    ([300], [301], 0, 1, 20, 48, 48, INTER, 1024, 1024),          # 40 rows, two workgroups of them
    ([5] * 70, list(range(5, 75)), 0, 2, 1, 112, 112, INTER, 16, 16)])
def test_append(ctx, name, q_lens, own_lens, prefix, heads, kv_heads, head_dim, rot, layout, page, block):
    _case(ctx, q_lens, own_lens, prefix, heads, kv_heads, head_dim, rot, layout, page, block, name)


def test_without_queries_without_rotation_and_other_orders(ctx):
    _case(ctx, [3, 1], [20, 9], 4, 0, 2, 64, 64, HALF, 16, 16, "bf16", order="slots")
    _case(ctx, [3, 1], [20, 9], 4, 3, 3, 64, 0, HALF, 32, 16, "f32", order="slots")
    _case(ctx, [40], [45], 0, 0, 1, 48, 10, INTER, 64, 64, "f16", order="slots")
    _case(ctx, [3, 1], [20, 9], 4, 4, 3, 64, 64, HALF, 32, 16, "bf16", order="major")


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("head_dim,rot,layout,page", [(128, 128, HALF, 64), (64, 32, INTER, 16), (48, 10, HALF, 32)])
def test_the_longest_sequence_is_only_a_hint(ctx, name, head_dim, rot, layout, page):
    # by tokens of a sequence a row of a block is one wave's or all waves'; every hint gives the same cache
    seen = []
    for max_q in (0, 1, 3, 100, 100000):
        p = Paged8([1, 70, 5, 33], [30, 90, 5, 40], 7, 3, head_dim, page, page, seed=4)
        g = torch.Generator(device="cuda").manual_seed(5)
        x = torch.randn(p.tokens, 2 * 3 + 5, head_dim, generator=g, device="cuda").to(TYPES[name])
        q, k, v = x.split([5, 3, 3], 1)
        out = torch.full((p.tokens, 5, head_dim), 7.0, dtype=x.dtype, device="cuda")
        _append(ctx, p, vtq.Rope(rot, layout), name, k, v, q, out, desc=p.describe(max_q=max_q))
        seen.append([t.clone() for t in (p.dk, p.dv, p.dks, p.dvs, out.view(torch.uint8))])
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("name,head_dim,rot,layout,block", [("f32", 128, 0, HALF, 64), ("bf16", 256, 256, HALF, 32),
                                                            ("f16", 64, 32, INTER, 128), ("f32", 48, 10, HALF, 64)])
def test_long_blocks_grow(ctx, seed, name, head_dim, rot, layout, block):
    # rows of a block that all waves of a workgroup share, behind tokens that are quieter or louder
    _case(ctx, [30, 50, 1, 7], [40, 61, 9, 130], 3, 4, 2, head_dim, rot, layout, 128, name=name, block=block, seed=seed,
          loud=4.0)


@pytest.mark.parametrize("seed", range(4))
def test_scales_grow_and_stay(ctx, seed):
    # tokens louder and quieter than those before them in the block, by up to some powers of two
    _case(ctx, [1] * 12, [2 + i for i in range(12)], 0, 0, 2, 64, 0, HALF, 32, 32, "f32", seed=seed, loud=4.0)
    _case(ctx, [5] * 6, [6, 9, 12, 17, 20, 31], 3, 2, 2, 32, 32, INTER, 32, 32, "f32", seed=seed, loud=6.0)


def test_any_byte_of_a_scale_is_a_scale(ctx):
    def bytes_(p):
        for b, byte in enumerate((0, 1, 9, 10, 246, 247, 255)):
            p.ks[int(p.pages[b, 0])] = byte
            p.vs[int(p.pages[b, 0])] = byte

    _case(ctx, [1] * 7, [5] * 7, 0, 0, 2, 32, 0, HALF, 16, 16, "f32", change=bytes_)


def test_extreme_values(ctx):
    for scale in (1e-45, 1e-38, 3e-36, 1e30, 3e38):
        p = Paged8([4, 1], [4, 20], 0, 1, 32, 16)
        x = torch.randn(5, 2, 32).clamp(-1, 1) * scale
        x[1, 0, 3], x[2, 0, 4], x[4, 1, 5] = float("inf"), float("nan"), -float("inf")
        x[3] = 0.0
        dev = x.cuda()
        k, v = dev.split([1, 1], 1)
        _append(ctx, p, None, "f32", k, v)
        _check(p, x, 0, 0, HALF, "f32")
    # a block of zeros, and one of nothing finite: the least scale
    p = Paged8([2, 2], [2, 2], 0, 1, 16, 16)
    x = torch.zeros(4, 2, 16)
    x[2:] = float("nan")
    dev = x.cuda()
    _append(ctx, p, None, "f32", dev[:, :1], dev[:, 1:])
    _check(p, x, 0, 0, HALF, "f32")
    assert int(p.dks.cpu()[int(p.pages[0, 0]), 0, 0]) == 10


def test_the_largest_element_at_a_border_of_scales(ctx):
    # 448 * 2^e takes e, the next f32 number e + 1
    p = Paged8([1] * 4, [1] * 4, 0, 1, 16, 16)
    x = torch.ones(4, 2, 16)
    x[0, :, 3] = 448.0 * 2.0 ** -7
    x[1, :, 3] = torch.nextafter(torch.tensor(448.0 * 2.0 ** -7), torch.tensor(10.0))
    x[2, :, 3] = -448.0
    x[3, :, 3] = 512.0
    dev = x.cuda()
    _append(ctx, p, None, "f32", dev[:, :1], dev[:, 1:])
    _check(p, x, 0, 0, HALF, "f32")
    got = [int(p.dks.cpu()[int(p.pages[b, 0]), 0, 0]) - 127 for b in range(4)]
    assert got == [-7, -6, 0, 1]


def test_rows_behind_the_last_sequence_stay(ctx):
    _case(ctx, [3, 2], [8, 8], 0, 4, 2, 64, 64, HALF, 16, 16, "bf16", spare_tokens=5)


def test_tokens_without_a_slot_are_not_written_and_scale_nothing(ctx):
    # a sequence shorter than its new tokens: the ones before place 0 are loud
    p = Paged8([4, 3], [2, 16], 10, 2, 64, 16)
    x = torch.randn(7, 4, 64)
    x[:2] *= 1e6
    dev = x.cuda()
    _append(ctx, p, None, "f32", dev[:, :2], dev[:, 2:])
    _check(p, x, 0, 0, HALF, "f32")
    p = Paged8([3, 2, 2], [18, 40, 5], 0, 2, 64, 16, fill=False)
    p.pages[0, 1], p.pages[1, 2], p.pages[2, 0] = -1, p.n_pages, 2 ** 31 - 1
    p.len[2] = 16 * p.max_pages + 2  # both new tokens past the list
    p.own_lens[2] = 16 * p.max_pages + 2
    p.to_device()
    x[:3] *= 100.0
    dev = x.cuda()
    _append(ctx, p, None, "f32", dev[:, :2], dev[:, 2:])
    _check(p, x, 0, 0, HALF, "f32")
    # the slots before it are of its block: NaNs, which a larger scale leaves NaNs of either sign
    changed = (p.dk.cpu() != p.kc).any(-1).any(1)  # [pages, slots]
    assert set(changed.nonzero()[:, 0].tolist()) == {int(p.pages[0, 0])} and changed[int(p.pages[0, 0]), 15]


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_token_by_token_and_at_once(ctx, name):
    # the last scale is the same either way; elements differ by what fell below the least normal value
    own, d, block = 45, 64, 32
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(own, 2, d, generator=g) * torch.exp2(torch.randn(own, 1, 1, generator=g))).to(TYPES[name])
    dev = x.cuda()
    once = Paged8([own], [own], 0, 1, d, 32, block, fill=False)
    _append(ctx, once, vtq.Rope(d), name, dev[:, :1], dev[:, 1:])
    step = Paged8([1], [own], 0, 1, d, 32, block, fill=False)
    for i in range(own):
        step.dlists[1].fill_(i + 1)
        _append(ctx, step, vtq.Rope(d), name, dev[i:i + 1, :1], dev[i:i + 1, 1:])
    once.from_device(), step.from_device()
    for a, b, scale in ((once.kh, step.kh, once.ks), (once.vh, step.vh, once.vs)):
        page = [int(p) for p in once.pages[0]]
        first = [int(p) for p in step.pages[0]]
        for j in range(-(-own // 32)):
            m = min(32, own - 32 * j)
            assert torch.equal(once.scale_view(once.ks)[page[j]], step.scale_view(step.ks)[first[j]])
            u, v = a[page[j], :, :m], b[first[j], :, :m]
            e = scale[page[j], :, 0].double()[:, None, None] - 127
            assert ((u - v).abs() <= E8_STEP * torch.exp2(e)).all()
            assert torch.equal(u[u.abs() >= 2.0 ** -5 * torch.exp2(e).expand_as(u)],
                               v[u.abs() >= 2.0 ** -5 * torch.exp2(e).expand_as(u)])


E8_STEP = 2.0 ** -9  # the step below the least normal value: halves of it from each of two roundings


def test_the_same_call_twice_changes_nothing_more(ctx):
    p, dev = _case(ctx, [3, 40], [20, 61], 7, 2, 2, 64, 64, HALF, 64, 32, "bf16", seed=9, loud=3.0)
    state = [t.clone() for t in (p.dk, p.dv, p.dks, p.dvs)]
    q, k, v = dev.split([2, 2, 2], 1)
    _append(ctx, p, vtq.Rope(64, HALF), "bf16", k, v, q, torch.empty_like(q))
    for a, b in zip(state, (p.dk, p.dv, p.dks, p.dvs)):
        assert torch.equal(a, b)


def test_unaligned_rows(ctx):
    # rows that start at odd elements: one element an access
    for name in ("f32", "bf16"):
        p = Paged8([5, 1], [20, 33], 0, 2, 32, 16)
        x = torch.randn(6, 6 * 32 + 1).to(TYPES[name])
        dev = x.cuda()
        rows = dev[:, 1:].unflatten(1, (6, 32))
        out = torch.empty(6, 2, 32, dtype=TYPES[name], device="cuda")
        _append(ctx, p, vtq.Rope(16, INTER), name, rows[:, 2:4], rows[:, 4:], rows[:, :2], out)
        _check(p, x[:, 1:].unflatten(1, (6, 32)), 2, 16, INTER, name)


def test_in_place_queries_and_a_replayed_graph(ctx):
    p = Paged8([1, 1, 1], [5, 17, 30], 9, 2, 128, 16)
    rope = vtq.Rope(128, HALF)
    q0 = torch.randn(3, 8, 128, device="cuda").bfloat16()
    k, v = (torch.randn(3, 2, 128, device="cuda").bfloat16() for _ in range(2))
    eager, q = torch.empty_like(q0), q0.clone()
    state = (p.dk, p.dv, p.dks, p.dvs)

    def step(dst):
        ctx.kv8_append_device(p.cache, p.desc, rope, vtq.BF16, 3, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                              v.stride(0), v.stride(1), stream(), heads=8, q_ptr=q.data_ptr(), q_token_stride=q.stride(0),
                              q_head_stride=q.stride(1), q_out_ptr=dst.data_ptr(), q_out_token_stride=dst.stride(0),
                              q_out_head_stride=dst.stride(1))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q)
    for i in range(4):  # the lengths move on in device memory
        p.dlists[1].fill_(6 + i)
        k.normal_().mul_(2.0 ** i)
        q.copy_(q0)
        before = [t.clone() for t in state]
        step(eager)
        torch.cuda.synchronize()
        want = [t.clone() for t in state]
        for t, old in zip(state, before):
            t.copy_(old)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, eager)
        for t, w in zip(state, want):
            assert torch.equal(t, w)
        assert not torch.equal(want[0], before[0])


def test_offsets_past_32_bits(ctx):
    d, page, n_pages = 64, 64, (1 << 32) // (64 * 64) + 100
    kc = torch.empty(n_pages, 1, page, d, dtype=torch.uint8, device="cuda")
    vc = torch.empty(n_pages, 1, page, d, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(2, n_pages, 1, page // 16, dtype=torch.uint8, device="cuda")
    pages = torch.tensor([[n_pages - 1, 3]], dtype=torch.int32, device="cuda")
    lists = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([49], dtype=torch.int32, device="cuda")
    cache = vtq.Kv8Cache(kc.data_ptr(), vc.data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), n_pages, page, 1, d)
    batch = vtq.KvBatch(1, lists[0].data_ptr(), lists[1].data_ptr(), pages.data_ptr(), 2)
    k, v = (torch.randn(1, 1, d, device="cuda").half() for _ in range(2))
    kc[-1].zero_(), vc[-1].zero_()
    ctx.kv8_append_device(cache, batch, None, vtq.F16, 1, k.data_ptr(), d, d, v.data_ptr(), d, d, stream())
    torch.cuda.synchronize()
    for c, s, x in ((kc, scales[0], k), (vc, scales[1], v)):
        e = int(s[-1, 0, 3]) - 127
        want = torch.ldexp(x[0, 0].float(), torch.tensor(-e, device="cuda")).to(torch.float8_e4m3fn).view(torch.uint8)
        assert same_codes(c[-1, 0, 48], want) and not c[-1, 0, :48].any() and not s[:-1].any()
