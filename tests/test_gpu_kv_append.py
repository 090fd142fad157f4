"""Appending to a paged cache with the rotation on the way (vtq_kv_append_device)."""
import pytest
import torch

import vtq
from serving import TAGS, TYPES, Paged, frequencies, rotate_exact, rotation_bound, stream, within

pytestmark = pytest.mark.gpu

HALF, INTER = vtq.ROPE_HALF, vtq.ROPE_INTERLEAVED


def _append(ctx, p, rope, name, k, v, q=None, out=None):
    args = {}
    if q is not None:
        args = dict(heads=q.shape[1], q_ptr=q.data_ptr(), q_token_stride=q.stride(0), q_head_stride=q.stride(1),
                    q_out_ptr=out.data_ptr(), q_out_token_stride=out.stride(0), q_out_head_stride=out.stride(1))
    ctx.kv_append_device(p.cache, p.desc, rope, TAGS[name], k.shape[0], k.data_ptr(), k.stride(0), k.stride(1),
                         v.data_ptr(), v.stride(0), v.stride(1), stream(), **args)
    torch.cuda.synchronize()


def _case(ctx, q_lens, own_lens, prefix, heads, kv_heads, head_dim, rot, layout, page, name, cache, order="heads",
          seed=0, spare_tokens=0):
    """Appends and compares the whole cache: the tokens' slots by bounds, every other one bit for bit."""
    p = Paged(q_lens, own_lens, prefix, kv_heads, head_dim, page, cache, seed=seed, layout=order)
    g = torch.Generator().manual_seed(seed + 1)
    tokens = p.tokens + spare_tokens
    packed = torch.randn(tokens, heads + 2 * kv_heads, head_dim, generator=g).to(TYPES[name])
    dev = packed.cuda()
    q, k, v = dev.split([heads, kv_heads, kv_heads], 1)
    out = torch.full((tokens, heads, head_dim), 7.0, dtype=q.dtype, device="cuda")
    rope = vtq.Rope(rot, layout) if rot else None
    before_k, before_v = p.dk.clone(), p.dv.clone()
    _append(ctx, p, rope, name, k, v, q if heads else None, out)
    where = p.places()
    pos = torch.tensor([prefix + place for _, place in where], dtype=torch.int64)
    freq, m = frequencies(rot) if rot else (torch.zeros(0, dtype=torch.float64), 1.0)
    want_q, size_q, _ = rotate_exact(packed[:p.tokens, :heads], pos, freq, m, layout)
    want_k, size_k, _ = rotate_exact(packed[:p.tokens, heads:heads + kv_heads], pos, freq, m, layout)
    want_v = packed[:p.tokens, heads + kv_heads:].to(TYPES[cache])
    if heads:
        within(out[:p.tokens], want_q, rotation_bound(want_q, size_q, q.dtype), "queries")
        assert (out[p.tokens:] == 7.0).all()
    bound_k = rotation_bound(want_k, size_k, TYPES[cache])
    got_k, got_v = p.dk.cpu(), p.dv.cpu()
    view_k, view_v, old_k, old_v = (p.view(t) for t in (got_k, got_v, before_k.cpu(), before_v.cpu()))
    for t, (b, place) in enumerate(where):
        if place < 0 or place // page >= p.max_pages or not 0 <= int(p.pages[b, place // page]) < p.n_pages:
            continue
        at = (int(p.pages[b, place // page]), slice(None), place % page)
        within(view_k[at], want_k[t], bound_k[t], f"key of token {t}")
        assert torch.equal(view_v[at], want_v[t]), f"value of token {t}"
        view_k[at], view_v[at] = old_k[at], old_v[at]
    assert torch.equal(view_k.view(torch.int32 if cache == "f32" else torch.int16),
                       old_k.view(torch.int32 if cache == "f32" else torch.int16))
    assert torch.equal(view_v.view(torch.int32 if cache == "f32" else torch.int16),
                       old_v.view(torch.int32 if cache == "f32" else torch.int16))


@pytest.mark.parametrize("name,cache", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"),
                                        ("f32", "bf16")])
@pytest.mark.parametrize("q_lens,own_lens,prefix,heads,kv_heads,head_dim,rot,layout,page", [
    ([1], [1], 0, 1, 1, 8, 8, HALF, 8),
    ([1] * 5, [1, 16, 17, 300, 64], 2000, 32, 8, 128, 128, HALF, 16),
    ([3, 0, 7, 1, 0], [3, 9, 40, 1, 0], 77, 4, 4, 64, 32, INTER, 32),
    ([40, 17], [40, 100], 0, 7, 1, 80, 80, HALF, 64),
    ([130], [130], 5, 6, 2, 96, 24, INTER, 16),
    ([2, 2], [5, 4097], 1, 8, 8, 256, 64, HALF, 4096),
    ([5] * 70, list(range(5, 75)), 0, 2, 1, 72, 72, INTER, 8)])
def test_append(ctx, name, cache, q_lens, own_lens, prefix, heads, kv_heads, head_dim, rot, layout, page):
    _case(ctx, q_lens, own_lens, prefix, heads, kv_heads, head_dim, rot, layout, page, name, cache)


def test_without_queries_without_rotation_and_slots_before_heads(ctx):
    _case(ctx, [3, 1], [20, 9], 4, 0, 2, 64, 64, HALF, 16, "bf16", "bf16", order="slots")
    _case(ctx, [3, 1], [20, 9], 4, 3, 3, 64, 0, HALF, 16, "f32", "f16", order="slots")
    _case(ctx, [2], [2], 0, 0, 1, 40, 10, INTER, 8, "f32", "f32", order="slots")
    _case(ctx, [3, 1], [20, 9], 4, 4, 3, 64, 64, HALF, 16, "bf16", "bf16", order="major")


def test_rows_behind_the_last_sequence_stay(ctx):
    _case(ctx, [3, 2], [8, 8], 0, 4, 2, 64, 64, HALF, 16, "bf16", "bf16", spare_tokens=5)


def test_tokens_without_a_slot_are_not_written(ctx):
    # a sequence shorter than its new tokens (places below 0) and one longer than its page list
    _case(ctx, [4, 3], [2, 16], 10, 2, 2, 64, 64, HALF, 16, "f32", "f32")
    p = Paged([3, 2, 2], [18, 40, 5], 0, 2, 64, 16, "bf16", fill=False)
    p.pages[0, 1], p.pages[1, 2], p.pages[2, 0] = -1, p.n_pages, 2 ** 31 - 1
    p.len[2] = 16 * p.max_pages + 2  # both new tokens past the list
    p.to_device()
    k = torch.randn(7, 2, 64, device="cuda").bfloat16()
    before = p.dk.clone()
    _append(ctx, p, vtq.Rope(64), "bf16", k, k)
    changed = (p.dk.view(torch.int16) != before.view(torch.int16)).any(-1).any(1)  # [pages, slots]
    # only place 15 of sequence 0 has a slot (16 and 17 are in page -1; 38, 39 of sequence 1 in page n_pages)
    assert changed.nonzero().tolist() == [[int(p.pages[0, 0]), 15]]


def test_in_place_queries_and_a_replayed_graph(ctx):
    p = Paged([1, 1, 1], [5, 17, 30], 9, 2, 128, 16, "bf16")
    rope = vtq.Rope(128, HALF)
    q0 = torch.randn(3, 8, 128, device="cuda").bfloat16()
    k, v = (torch.randn(3, 2, 128, device="cuda").bfloat16() for _ in range(2))
    eager = torch.empty_like(q0)
    q = q0.clone()

    def step(dst):
        ctx.kv_append_device(p.cache, p.desc, rope, vtq.BF16, 3, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                             v.stride(0), v.stride(1), stream(), heads=8, q_ptr=q.data_ptr(), q_token_stride=q.stride(0),
                             q_head_stride=q.stride(1), q_out_ptr=dst.data_ptr(), q_out_token_stride=dst.stride(0),
                             q_out_head_stride=dst.stride(1))

    step(eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q)
    for i in range(3):  # the lengths move on in device memory
        p.dlists[1].fill_(6 + i)
        q.copy_(q0)
        step(eager)
        want_k = p.dk.clone()
        p.dk.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, eager)
        for b in range(3):
            page = int(p.pages[b, 0])
            assert torch.equal(p.dk[page, :, 5 + i], want_k[page, :, 5 + i])
        p.dk.copy_(want_k)


def test_offsets_past_32_bits(ctx):
    # a cache of 2^32 + elements: the last pages lie behind 4 GiB and 2^31 elements
    d, page, n_pages = 64, 64, (1 << 31) // (64 * 64) + 100
    kc = torch.empty(n_pages, 1, page, d, dtype=torch.float16, device="cuda")
    vc = torch.empty(n_pages, 1, page, d, dtype=torch.float16, device="cuda")
    pages = torch.tensor([[n_pages - 1, 3]], dtype=torch.int32, device="cuda")
    lists = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([64], dtype=torch.int32, device="cuda")
    cache = vtq.KvCache(vtq.F16, kc.data_ptr(), vc.data_ptr(), n_pages, page, 1, d)
    batch = vtq.KvBatch(1, lists[0].data_ptr(), lists[1].data_ptr(), pages.data_ptr(), 2)
    k, v = (torch.randn(1, 1, d, device="cuda").half() for _ in range(2))
    kc[-1].zero_(), vc[-1].zero_()
    ctx.kv_append_device(cache, batch, None, vtq.F16, 1, k.data_ptr(), d, d, v.data_ptr(), d, d, stream())
    assert torch.equal(kc[-1, 0, 63], k[0, 0]) and torch.equal(vc[-1, 0, 63], v[0, 0]) and not kc[-1, 0, :63].any()
