"""Decoding with beams over an 8-bit cache, the operators together: projections, append, attention behind a shared
prefix, selection, the next step's page tables and the copies of part-filled pages, over two layers and several pages.
The beams that are left give the same cache, bit for bit, as the same tokens without a fork; the selections are checked
against 64 bits, the page counts against the tables, and a captured step against the eager ones."""
import math

import pytest
import torch

import vtq
from kv8 import Paged8, attention8_exact
from serving import TAGS, TYPES, stream, up16, within

pytestmark = pytest.mark.gpu

LAYERS, GROUPS, BEAMS, DIM, HEADS, KV_HEADS, HEAD_DIM, VOCAB, PAGE = 2, 3, 4, 96, 8, 2, 64, 257, 16
ROWS, MAX_PAGES, N_PAGES, PREFIX, END = GROUPS * BEAMS, 4, 80, 40, 11


class Decoder:
    """`ROWS` sequences, one token each a step.  The first layer's keys of the prefix are random; forks and ends follow
    `choose`, or without it the tokens are given."""

    def __init__(self, ctx, name, seed=0):
        self.ctx, self.name, self.tag = ctx, name, TAGS[name]
        g = torch.Generator(device="cuda").manual_seed(seed)
        dev = dict(device="cuda")
        rnd = lambda *s: torch.randn(*s, generator=g, **dev)  # noqa: E731
        self.embed = rnd(VOCAB, DIM).to(TYPES[name])
        qkv_rows = (HEADS + 2 * KV_HEADS) * HEAD_DIM
        self.w_qkv = [self.weights(rnd(qkv_rows, DIM) * 0.2) for _ in range(LAYERS)]
        self.w_out = [self.weights(rnd(DIM, HEADS * HEAD_DIM) * 0.1) for _ in range(LAYERS)]
        self.w_vocab = self.weights(rnd(VOCAB, DIM) * 0.4)
        self.x = torch.zeros(ROWS, DIM, dtype=TYPES[name], **dev)
        self.qkv = torch.zeros(ROWS, HEADS + 2 * KV_HEADS, HEAD_DIM, dtype=TYPES[name], **dev)
        self.a = torch.zeros(ROWS, HEADS * HEAD_DIM, dtype=TYPES[name], **dev)
        self.o = torch.zeros(ROWS, DIM, dtype=TYPES[name], **dev)
        self.logits = torch.zeros(ROWS, VOCAB + 3, dtype=TYPES[name], **dev)
        self.rope = vtq.Rope(HEAD_DIM, vtq.ROPE_HALF, theta=10000.0)
        # the layers' caches side by side; pages 0 to 2 are the prefix's
        shape = (LAYERS, N_PAGES, KV_HEADS, PAGE, HEAD_DIM)
        self.k, self.v = (torch.full(shape, 0x7F, dtype=torch.uint8, **dev) for _ in range(2))
        self.ks, self.vs = (torch.randint(0, 256, shape[:3] + (1,), generator=g, dtype=torch.uint8, **dev) for _ in range(2))
        n_prefix = -(-PREFIX // PAGE)
        for l in range(LAYERS):
            for codes, scale in ((self.k, self.ks), (self.v, self.vs)):
                x = rnd(n_prefix, KV_HEADS, PAGE, HEAD_DIM).clamp(-3, 3) * 100
                codes[l, :n_prefix] = x.to(torch.float8_e4m3fn).view(torch.uint8)
                codes[l, n_prefix - 1, :, PREFIX % PAGE:] = 0x7F
                scale[l, :n_prefix] = 127 - 6
        self.prefix_pages = torch.arange(n_prefix, dtype=torch.int32, **dev)
        self.q_start = torch.arange(ROWS + 1, dtype=torch.int32, **dev)
        # every sequence begins with one page of its own
        ints = lambda x: torch.tensor(x, dtype=torch.int32, **dev)  # noqa: E731
        self.refs = ints([1] * (n_prefix + ROWS) + [0] * (N_PAGES - n_prefix - ROWS))
        self.table = ints([[n_prefix + r] + [-1] * (MAX_PAGES - 1) for r in range(ROWS)])
        self.len, self.grow = ints([1] * ROWS), ints([1] * ROWS)
        self.token = ints([1 + r // BEAMS for r in range(ROWS)])
        self.score = torch.tensor([0.0] + [-math.inf] * (BEAMS - 1), **dev).repeat(GROUPS)
        self.done = torch.zeros(ROWS, dtype=torch.uint8, **dev)
        self.parent, self.copies, self.info = ints([0] * ROWS), ints([[0] * 3] * ROWS), ints([0, 0])
        self.new_refs, self.new_table, self.new_len = (torch.zeros_like(t) for t in (self.refs, self.table, self.len))
        self.batch = vtq.KvBatch(ROWS, self.q_start.data_ptr(), self.len.data_ptr(), self.table.data_ptr(), MAX_PAGES,
                                 prefix_len=PREFIX, prefix_pages=self.prefix_pages.data_ptr())
        self.caches = [vtq.Kv8Cache(*(t[l].data_ptr() for t in (self.k, self.v, self.ks, self.vs)), N_PAGES, PAGE, KV_HEADS,
                                    HEAD_DIM) for l in range(LAYERS)]
        need = (ctx.kv8_attention_workspace(self.caches[0], self.batch, self.tag, ROWS, HEADS),
                ctx.beam_select_workspace(GROUPS, BEAMS, VOCAB, BEAMS), ctx.pages_reorder_workspace(N_PAGES, ROWS, ROWS))
        self.ws = [torch.full((max(256, n),), 255, dtype=torch.uint8, **dev) for n in need]

    def weights(self, w):
        n, k = w.shape
        q, s = torch.zeros(n, up16(k), dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
        self.ctx.quantize_i8_device(vtq.F32, w.data_ptr(), k, q.data_ptr(), up16(k), s.data_ptr(), n, k, stream())
        return q, s, torch.zeros(ROWS, up16(k), dtype=torch.int8, device="cuda"), torch.zeros(ROWS, device="cuda")

    def linear(self, x, weights, y, n):
        q, s, x8, xs = weights
        k = x.shape[1]
        self.ctx.quantize_i8_device(self.tag, x.data_ptr(), k, x8.data_ptr(), x8.shape[1], xs.data_ptr(), ROWS, k, stream())
        self.ctx.linear_i8_device(x8.data_ptr(), x8.shape[1], xs.data_ptr(), q.data_ptr(), q.shape[1], s.data_ptr(), None,
                                  self.tag, y.data_ptr(), y.stride(0), ROWS, k, n, stream())

    def forward(self):
        torch.index_select(self.embed, 0, self.token, out=self.x)
        for l, cache in enumerate(self.caches):
            self.linear(self.x, self.w_qkv[l], self.qkv, (HEADS + 2 * KV_HEADS) * HEAD_DIM)
            q, k, v = self.qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
            at = (self.qkv.stride(0), self.qkv.stride(1))
            self.ctx.kv8_append_device(cache, self.batch, self.rope, self.tag, ROWS, k.data_ptr(), *at, v.data_ptr(), *at,
                                       stream(), heads=HEADS, q_ptr=q.data_ptr(), q_token_stride=at[0],
                                       q_head_stride=at[1], q_out_ptr=q.data_ptr(), q_out_token_stride=at[0],
                                       q_out_head_stride=at[1])
            self.ctx.kv8_attention_device(cache, self.batch, self.tag, ROWS, HEADS, q.data_ptr(), *at, self.a.data_ptr(),
                                          HEADS * HEAD_DIM, HEAD_DIM, HEAD_DIM**-0.5, self.ws[0].data_ptr(),
                                          self.ws[0].numel(), stream())
            self.linear(self.a, self.w_out[l], self.o, DIM)
            torch.add(self.x, self.o, out=self.x)
        self.linear(self.x, self.w_vocab, self.logits, VOCAB)

    def choose(self):
        c = self.ctx
        c.beam_select_device(self.tag, self.logits.data_ptr(), self.logits.stride(0), GROUPS, BEAMS, VOCAB,
                             self.score.data_ptr(), BEAMS, self.score.data_ptr(), self.token.data_ptr(),
                             self.parent.data_ptr(), self.ws[1].data_ptr(), self.ws[1].numel(), stream(),
                             done_ptr=self.done.data_ptr(), end_token=END, out_done_ptr=self.done.data_ptr())
        c.pages_reorder_device(N_PAGES, PAGE, MAX_PAGES, self.refs.data_ptr(), ROWS, self.table.data_ptr(),
                               self.len.data_ptr(), ROWS, self.parent.data_ptr(), self.grow.data_ptr(),
                               self.new_refs.data_ptr(), self.new_table.data_ptr(), self.new_len.data_ptr(),
                               self.copies.data_ptr(), self.info.data_ptr(), self.ws[2].data_ptr(), self.ws[2].numel(),
                               stream())
        c.pages_copy_device(self.caches[0], LAYERS, self.k.stride(0), self.copies.data_ptr(), ROWS, self.info.data_ptr(),
                            stream(), scale_layer_stride=self.ks.stride(0))
        torch.add(self.new_refs, 0, out=self.refs)
        torch.add(self.new_table, 0, out=self.table)
        torch.add(self.new_len, 1, out=self.len)

    def state(self):
        return [t.clone() for t in (self.refs, self.table, self.len, self.token, self.parent, self.score, self.done,
                                    self.k, self.v, self.ks, self.vs, self.logits, self.info)]


def _best(logits, score, done):
    """[(sum, row, token)] of each group, from 64 bits."""
    x = logits[:, :VOCAB].double().cpu()
    s = score.double().cpu()[:, None] + x - x.logsumexp(1, keepdim=True)
    out = []
    for g in range(GROUPS):
        some = []
        for r in range(g * BEAMS, (g + 1) * BEAMS):
            if done[r]:
                some.append((-float(score[r]), 0.0, r, END))
            else:
                some += [(-float(s[r, t]), -float(x[r, t]), r, t) for t in range(VOCAB)]
        out += [(-a, r, t) for a, _, r, t in sorted(some)[:BEAMS]]
    return out


def _no_forks(ctx, name, tokens):
    """A decoder whose ROWS sequences took these tokens [steps][row] one after another, with pages as they need them."""
    d = Decoder(ctx, name)
    n_prefix = len(d.prefix_pages)
    for t, row in enumerate(tokens):
        if t % PAGE == 0:
            d.table[:, t // PAGE] = n_prefix + torch.arange(ROWS, dtype=torch.int32, device="cuda") + t // PAGE * ROWS
        d.len.fill_(t + 1)
        d.token.copy_(torch.tensor(row, dtype=torch.int32))
        d.forward()
    return d


@pytest.mark.parametrize("name,steps", [("f32", 37), ("bf16", 50), ("f16", 20)])
def test_beams_over_an_8_bit_cache(ctx, name, steps):
    d = Decoder(ctx, name)
    history = [[] for _ in range(ROWS)]  # the tokens that each sequence's cache holds
    copies = 0
    for step in range(steps):
        inputs = d.token.tolist()
        history = [h + [t] for h, t in zip(history, inputs)]
        d.forward()
        if step in (0, 17, steps - 1):
            # the last layer's attention against 64 bits, on the queries and the cache that it read
            p = Paged8([1] * ROWS, [step + 1] * ROWS, PREFIX, KV_HEADS, HEAD_DIM, PAGE, device=None, fill=False)
            p.n_pages, p.max_pages = N_PAGES, MAX_PAGES
            p.kc, p.vc, p.ks, p.vs = (t[-1].cpu() for t in (d.k, d.v, d.ks, d.vs))
            p.pages, p.prefix_pages = d.table.cpu().clamp(min=0), d.prefix_pages.cpu()
            p.refresh()
            q = d.qkv[:, :HEADS].cpu()
            want, _, by, _ = attention8_exact(p, q, HEADS, HEAD_DIM**-0.5)
            within(d.a.view(ROWS, HEADS, HEAD_DIM), want, by, f"attention of step {step}")
        want = _best(d.logits, d.score, d.done.tolist())
        was_done = d.done.tolist()
        d.choose()
        torch.cuda.synchronize()
        got = list(zip(d.score.tolist(), d.parent.tolist(), d.token.tolist()))
        assert [x[1:] for x in got] == [x[1:] for x in want], step
        for (a, _, _), (b, _, _) in zip(got, want):
            assert a == b or abs(a - b) <= 2**-23 * abs(b) + 2**-30
        parents = d.parent.tolist()
        assert d.done.tolist() == [int(was_done[p] or t == END) for p, t in zip(parents, d.token.tolist())]
        history = [history[p] for p in parents]
        assert int(d.info[1]) == 0
        copies += int(d.info[0])
        # every page's count is that of the rows that name it; the prefix keeps its own
        held = torch.zeros(N_PAGES, dtype=torch.int64)
        held[:len(d.prefix_pages)] = 1
        for row in d.table.tolist():
            for page in row:
                if page >= 0:
                    held[page] += 1
        assert d.refs.tolist() == held.tolist()
        assert d.len.tolist() == [step + 2] * ROWS
    assert copies > 4  # forks within a page happened
    # the same tokens without forks
    serial = _no_forks(ctx, name, list(zip(*history)))
    for r in range(ROWS):
        for place in range(steps):
            a, b = int(d.table[r, place // PAGE]), int(serial.table[r, place // PAGE])
            for mine, other, one in ((d.k, serial.k, True), (d.v, serial.v, True), (d.ks, serial.ks, False),
                                     (d.vs, serial.vs, False)):
                x, y = mine[:, a], other[:, b]
                if one:
                    x, y = x[:, :, place % PAGE], y[:, :, place % PAGE]
                assert torch.equal(x, y), (r, place, one)


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_a_captured_step_of_beams(ctx, name):
    eager, d = Decoder(ctx, name, seed=3), Decoder(ctx, name, seed=3)
    states = []
    for _ in range(21):
        eager.forward()
        eager.choose()
        states.append(eager.state())
    start = d.state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # once before, so that libraries have what they allocate
        d.forward()
        d.choose()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for t, s in zip((d.refs, d.table, d.len, d.token, d.parent, d.score, d.done, d.k, d.v, d.ks, d.vs, d.logits, d.info),
                    start):
        t.copy_(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d.forward()
        d.choose()
    for step, want in enumerate(states):
        graph.replay()
        if step % 5 == 0:
            torch.cuda.synchronize()
            (torch.ones(1000, device="cuda") * step).sum().item()  # eager work between the replays
        for i, (a, b) in enumerate(zip(d.state(), want)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), (step, i)
