"""The serving operators together, as a step of a batch uses them: int8 q|k|v product, rotation and append, attention
over the shared prefix, int8 output product.  Each stage is checked against 64 bits on what the stage before gave (a
whole step's error would depend on which way an activation's rounding to 8 bits fell), and a captured step that
follows the lengths in device memory gives the eager steps' bits."""
import math

import pytest
import torch

import vtq
from serving import (F32_HALF_STEP, Paged, TAGS, TYPES, attention_exact, frequencies, half_step, quantize_exact,
                     rotate_exact, rotation_bound, smallest, stream, up16, within)

pytestmark = pytest.mark.gpu


class Layer:
    """One attention block: dim inputs, heads x head_dim queries, kv_heads keys and values."""

    def __init__(self, ctx, p, dim, heads, name, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.p, self.dim, self.heads, self.name = ctx, p, dim, heads, name
        d, hk = p.head_dim, p.kv_heads
        self.rows = (heads + 2 * hk) * d
        self.rope = vtq.Rope(d, vtq.ROPE_HALF, theta=500000.0)
        t = p.q_capacity
        dev = dict(device="cuda")
        self.wq, self.ws = self.weights(self.rows, dim, g)
        self.oq, self.os = self.weights(dim, heads * d, g)
        self.x = torch.randn(t, dim, generator=g, **dev).to(TYPES[name])
        self.x8, self.xs = torch.zeros(t, up16(dim), dtype=torch.int8, **dev), torch.zeros(t, **dev)
        self.qkv = torch.zeros(t, heads + 2 * hk, d, dtype=TYPES[name], **dev)
        self.a = torch.zeros(t, heads, d, dtype=TYPES[name], **dev)
        self.a8, self.as_ = torch.zeros(t, up16(heads * d), dtype=torch.int8, **dev), torch.zeros(t, **dev)
        self.y = torch.zeros(t, dim, dtype=TYPES[name], **dev)

    def weights(self, out_feat, in_feat, g):
        w = torch.randn(out_feat, in_feat, generator=g, device="cuda") * 0.05
        q = torch.zeros(out_feat, up16(in_feat), dtype=torch.int8, device="cuda")
        s = torch.zeros(out_feat, device="cuda")
        self.ctx.quantize_i8_device(vtq.F32, w.data_ptr(), in_feat, q.data_ptr(), up16(in_feat), s.data_ptr(), out_feat,
                                    in_feat, stream())
        return q, s

    def linear(self, x, x8, xs, wq, ws, y, tokens):
        tag, n, k = TAGS[self.name], y.numel() // y.shape[0], x.numel() // x.shape[0]
        self.ctx.quantize_i8_device(tag, x.data_ptr(), k, x8.data_ptr(), x8.shape[1], xs.data_ptr(), tokens, k, stream())
        self.ctx.linear_i8_device(x8.data_ptr(), x8.shape[1], xs.data_ptr(), wq.data_ptr(), wq.shape[1], ws.data_ptr(),
                                  None, tag, y.data_ptr(), n, tokens, k, n, stream())

    def step(self, desc, tokens, ws):
        p, tag, d = self.p, TAGS[self.name], self.p.head_dim
        q, k, v = self.qkv.split([self.heads, p.kv_heads, p.kv_heads], 1)
        self.linear(self.x, self.x8, self.xs, self.wq, self.ws, self.qkv, tokens)
        self.ctx.kv_append_device(p.cache, desc, self.rope, tag, tokens, k.data_ptr(), k.stride(0), k.stride(1),
                                  v.data_ptr(), v.stride(0), v.stride(1), stream(), heads=self.heads, q_ptr=q.data_ptr(),
                                  q_token_stride=q.stride(0), q_head_stride=q.stride(1), q_out_ptr=q.data_ptr(),
                                  q_out_token_stride=q.stride(0), q_out_head_stride=q.stride(1))
        self.ctx.attention_device(p.cache, desc, tag, tokens, self.heads, q.data_ptr(), q.stride(0), q.stride(1),
                                  self.a.data_ptr(), self.a.stride(0), self.a.stride(1), 1.0 / math.sqrt(d),
                                  ws.data_ptr(), ws.numel(), stream())
        self.linear(self.a, self.a8, self.as_, self.oq, self.os, self.y, tokens)


def _check_linear(x, x8, xs, wq, ws, y, tokens, what):
    k, n = x.numel() // x.shape[0], y.numel() // y.shape[0]
    want_q, want_s = quantize_exact(x[:tokens].reshape(tokens, k).cpu())
    assert torch.equal(x8[:tokens, :k].cpu(), want_q) and torch.equal(xs[:tokens].cpu(), want_s), what
    want = want_q.double() @ wq[:, :k].cpu().double().t() * want_s.double()[:, None] * ws.cpu().double()[None]
    bound = 4.01 * F32_HALF_STEP * want.abs() + half_step(y.dtype) * want.abs() * (1 + 1e-6) + smallest(y.dtype)
    within(y[:tokens].reshape(tokens, n), want, bound, what)


@pytest.mark.parametrize("name,cache", [("bf16", "bf16"), ("f32", "f16"), ("f32", "f32")])
def test_prompts_then_decoding(ctx, name, cache):
    prefix, heads, kv_heads, d, dim = 100, 8, 2, 64, 320
    lens = [37, 5, 60]
    p = Paged(lens, lens, prefix, kv_heads, d, 16, cache, extra_pages=1)
    p.q_capacity = sum(lens)
    layer = Layer(ctx, p, dim, heads, name, seed=1)
    descs = {"prompt": p.describe(max(lens)), "decode": p.describe(1)}
    need = max(ctx.attention_workspace(p.cache, x, TAGS[name], n, heads)
               for x, n in ((descs["prompt"], sum(lens)), (descs["decode"], 3)))
    ws = torch.zeros(need + 16, dtype=torch.uint8, device="cuda")
    layer.step(descs["prompt"], sum(lens), ws)
    torch.cuda.synchronize()
    _verify(p, layer, sum(lens))
    # one token of each sequence a step: the lists in device memory move on
    p.q_lens = [1, 1, 1]
    p.q_start.copy_(torch.tensor([0, 1, 2, 3]))
    p.tokens = 3
    p.dlists[0].copy_(p.q_start)
    graph = None
    for i in range(4):
        p.own_lens = [n + 1 for n in p.own_lens]
        p.dlists[1].add_(1)
        layer.x.copy_(torch.randn(layer.x.shape, device="cuda"))
        layer.step(descs["decode"], 3, ws)
        torch.cuda.synchronize()
        _verify(p, layer, 3)
        eager = [t.clone() for t in (layer.y, layer.a, layer.qkv, p.dk, p.dv)]
        if graph is None:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                layer.step(descs["decode"], 3, ws)
        # the step again from the graph: the same slots, the same bits
        for t in (layer.y, layer.a, layer.qkv):
            t.fill_(float("nan"))
        for t in (p.dk, p.dv):
            for b, n in enumerate(p.own_lens):
                page = int(p.pages[b, (n - 1) // 16])
                t[page, :, (n - 1) % 16].zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((layer.y, layer.a, layer.qkv), eager):
            assert torch.equal(got[:3], want[:3]) and got[3:].isnan().all()
        for got, want in zip((p.dk, p.dv), eager[3:]):
            bits = torch.int32 if cache == "f32" else torch.int16
            assert torch.equal(got.view(bits), want.view(bits))


def _verify(p, layer, tokens):
    heads, hk, d = layer.heads, p.kv_heads, p.head_dim
    # q|k|v before the rotation: the product again, elsewhere
    plain = torch.zeros_like(layer.qkv)
    layer.linear(layer.x, layer.x8, layer.xs, layer.wq, layer.ws, plain, tokens)
    torch.cuda.synchronize()
    _check_linear(layer.x, layer.x8, layer.xs, layer.wq, layer.ws, plain, tokens, "q|k|v")
    where = p.places()
    pos = torch.tensor([p.prefix + place for _, place in where])
    freq, m = frequencies(d, theta=500000.0)
    want_q, size_q, _ = rotate_exact(plain[:tokens, :heads], pos, freq, m, vtq.ROPE_HALF)
    want_k, size_k, _ = rotate_exact(plain[:tokens, heads:heads + hk], pos, freq, m, vtq.ROPE_HALF)
    within(layer.qkv[:tokens, :heads], want_q, rotation_bound(want_q, size_q, layer.qkv.dtype), "rotated queries")
    p.kh.copy_(p.dk.cpu())
    p.vh.copy_(p.dv.cpu())
    bound_k = rotation_bound(want_k, size_k, p.k.dtype)
    for t, (b, place) in enumerate(where):
        at = (int(p.pages[b, place // p.page]), slice(None), place % p.page)
        within(p.kh[at], want_k[t], bound_k[t], "cached key")
        assert torch.equal(p.vh[at], plain[t, heads + hk:].to(p.v.dtype).cpu())
    y, _, by, _ = attention_exact(p, layer.qkv[:tokens, :heads].cpu(), heads, float(torch.tensor(1.0 / math.sqrt(d))))
    within(layer.a[:tokens], y, by, "attention")
    _check_linear(layer.a, layer.a8, layer.as_, layer.oq, layer.os, layer.y, tokens, "output")
