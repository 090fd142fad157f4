"""Choosing the best continuations of beams (vtq_beam_select_device) against a sort in 64 bits."""
import numpy as np
import pytest
import torch

import vtq
from kv8 import log_softmax
from serving import F32_HALF_STEP, TAGS, TYPES, stream

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def _expect(x, score, groups, beams, n_out, done=None, end=-1):
    """(score in 64 bits, token, parent, done) of every output: candidates sorted by falling sum, falling logit, rising
    row and token.  x [rows, vocab] and score as numpy, in their stored values."""
    vocab = x.shape[1]
    out = []
    for g in range(groups):
        s, logit, row, token = [], [], [], []
        for r in range(g * beams, (g + 1) * beams):
            xr = x[r].astype(np.float64)
            if done is not None and done[r]:
                c = float(score[r])
                ok = np.isfinite(c)
                s.append(np.array([c if ok else -INF]))
                logit.append(np.array([0.0 if ok else -INF]))
                token.append(np.array([end]))
            else:
                top = xr.max()
                flat = not np.isfinite(score[r]) or np.isnan(xr).any() or not np.isfinite(top)
                if flat:
                    s.append(np.full(vocab, -INF))
                    logit.append(np.full(vocab, -INF))
                else:
                    s.append(float(score[r]) + log_softmax(xr[None])[0])
                    logit.append(xr)
                token.append(np.arange(vocab))
            row.append(np.full(len(s[-1]), r))
        s, logit, row, token = (np.concatenate(a) for a in (s, logit, row, token))
        order = np.lexsort((token, row, -logit, -s))[:n_out]
        got = [(s[i], int(token[i]), int(row[i]), int(bool(done is not None and done[row[i]]) or (0 <= end == token[i])))
               for i in order]
        out.append(got + [(-INF, -1, -1, 1)] * (n_out - len(got)))
    return out


def _select(ctx, x, score, groups, beams, n_out, done=None, end=-1, wait=True):
    name = next(k for k, t in TYPES.items() if t == x.dtype)
    vocab = x.shape[1]
    outs = (torch.full((groups, n_out), 7.0, device="cuda"), torch.full((groups, n_out), 7, dtype=torch.int32, device="cuda"),
            torch.full((groups, n_out), 7, dtype=torch.int32, device="cuda"),
            torch.full((groups, n_out), 7, dtype=torch.uint8, device="cuda"))
    need = ctx.beam_select_workspace(groups, beams, vocab, n_out)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    ctx.beam_select_device(TAGS[name], x.data_ptr(), x.stride(0), groups, beams, vocab, score.data_ptr(), n_out,
                           outs[0].data_ptr(), outs[1].data_ptr(), outs[2].data_ptr(), ws.data_ptr(), need, stream(),
                           done_ptr=None if done is None else done.data_ptr(), end_token=end,
                           out_done_ptr=outs[3].data_ptr())
    if wait:
        torch.cuda.synchronize()
        assert (ws[need:] == 255).all()
        return outs
    return outs, ws


def _check(outs, want, what=""):
    score, token, parent, done = (t.cpu() for t in outs)
    for g, rows in enumerate(want):
        for i, (s, t, p, d) in enumerate(rows):
            got = (int(token[g, i]), int(parent[g, i]), int(done[g, i]))
            assert got == (t, p, d), (what, g, i, got, (t, p, d), float(score[g, i]), s)
            # one rounding of a sum that is right to f64's last places (sums of 2^20 terms: 2^-40 of the largest)
            assert float(score[g, i]) == s or abs(float(score[g, i]) - s) <= F32_HALF_STEP * abs(s) * 1.001 + 1e-9, \
                (what, g, i, float(score[g, i]), s)


def _case(ctx, groups, beams, vocab, n_out, name, seed=0, spread=3.0, change=None, done=None, end=-1, pad=0, shift=0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(groups * beams, vocab, generator=g)).to(TYPES[name])
    score = -10.0 * torch.rand(groups * beams, generator=g)
    if change:
        change(x, score)
    wide = torch.full((groups * beams, vocab + pad + shift), NAN, dtype=x.dtype)
    wide[:, shift:shift + vocab] = x
    dev = wide.cuda()[:, shift:shift + vocab]
    d = None if done is None else torch.tensor(done, dtype=torch.uint8)
    outs = _select(ctx, dev, score.cuda(), groups, beams, n_out, None if d is None else d.cuda(), end)
    _check(outs, _expect(x.float().numpy(), score.numpy(), groups, beams, n_out, None if d is None else d.numpy(), end),
           (groups, beams, vocab, n_out, name, seed))
    return dev, score, outs


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab,n_out", [
    (1, 1, 1, 1), (1, 4, 32000, 8), (3, 2, 7, 5), (2, 5, 50257, 10), (1, 1, 2047, 64), (1, 1, 2049, 64), (2, 16, 999, 32),
    (1, 64, 500, 64), (5, 3, 8192, 6), (2, 3, 8193, 17), (1, 2, 130000, 4), (40, 4, 20000, 8), (70, 8, 9001, 16),
    (300, 2, 64, 3)])
def test_selection(ctx, name, groups, beams, vocab, n_out):
    _case(ctx, groups, beams, vocab, n_out, name, seed=vocab)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shift,pad", [(0, 5), (1, 0), (3, 2), (7, 9)])
def test_rows_at_any_element(ctx, name, shift, pad):
    _case(ctx, 2, 3, 5001, 6, name, shift=shift, pad=pad)
    _case(ctx, 180, 3, 8200, 6, name, shift=shift, pad=pad)  # 32 elements to a thread


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_out", [1, 16, 17, 64])
def test_all_alike(ctx, name, n_out):
    # every logit the same: the lowest rows and tokens
    def same(x, score):
        x.fill_(0.5)
        score.fill_(-2.0)

    _case(ctx, 2, 3, 5000, n_out, name, change=same)
    _case(ctx, 170, 3, 9000, n_out, name, change=same)
    _case(ctx, 1, 3, 20, n_out, name, change=same)


def test_equal_beams(ctx):
    # the first step: all beams alike but for their scores, or not even these
    def first(x, score):
        x.copy_(x[0].expand_as(x).clone())
        score.fill_(-1e9)
        score[0] = 0.0

    def alike(x, score):
        x.copy_(x[0].expand_as(x).clone())
        score.fill_(-1.5)

    def minus_infinity(x, score):
        first(x, score)
        score[1:] = -INF

    for change in (first, alike, minus_infinity):
        for n_out in (4, 8, 64):
            _case(ctx, 1, 8, 3001, n_out, "f32", change=change)
    _case(ctx, 1, 8, 3, 24, "f32", change=minus_infinity)  # masked beams' candidates fill the rest


@pytest.mark.parametrize("left", [0, 1, 3, 40, 300, 700])
def test_masked_tokens(ctx, left):
    # all but a few tokens at -infinity, or at the type's lowest number
    for lowest in (-INF, torch.finfo(torch.float32).min):
        for vocab, groups in ((5000, 2), (9000, 180)):
            def mask(x, score):
                g = torch.Generator().manual_seed(left)
                keep = torch.randperm(x.shape[1], generator=g)[:left]
                y = torch.full_like(x, lowest)
                y[:, keep] = x[:, keep]
                x.copy_(y)

            _case(ctx, groups, 3, vocab, 7, "f32", change=mask)
            _case(ctx, groups, 3, vocab, 40, "f32", change=mask)


def test_rows_that_are_no_numbers(ctx):
    def bad(x, score):
        x[0, 5], x[1, 9], x[2, :], x[3, 4] = NAN, INF, -INF, -INF
        score[5], score[6], score[7] = NAN, -INF, INF

    for n_out in (3, 16, 40):
        _case(ctx, 1, 10, 3000, n_out, "f32", change=bad)
        _case(ctx, 5, 2, 3000, n_out, "f32", change=bad)
        _case(ctx, 2, 5, 12, n_out, "f32", change=bad)

    def none(x, score):
        x[:, 0] = NAN

    _case(ctx, 2, 2, 100, 12, "f32", change=none)  # -infinities by row and token


def test_beams_that_ended(ctx):
    for n_out in (4, 8, 40):
        _case(ctx, 2, 4, 3000, n_out, "bf16", done=[1, 0, 0, 1, 0, 0, 0, 0], end=2)
        _case(ctx, 2, 4, 3000, n_out, "f32", done=[1, 1, 1, 1, 0, 1, 1, 1], end=0)   # fewer candidates than n_out
        _case(ctx, 2, 4, 5, n_out, "f32", done=[1, 1, 1, 1, 0, 1, 0, 1], end=-1)
    # an ended row's logits are not read, whatever they are

    def bad(x, score):
        x[1] = NAN

    _case(ctx, 1, 3, 1000, 6, "f32", done=[0, 7, 0], end=999, change=bad)
    # a row that ends now

    def likely(x, score):
        x[:, 2] = 30.0

    dev, score, outs = _case(ctx, 1, 2, 1000, 4, "f32", end=2, change=likely)
    assert outs[3].cpu()[0].tolist()[:2] == [1, 1]
    # an ended row of a score that is not finite
    def lost(x, score):
        score[0], score[1] = -INF, NAN

    _case(ctx, 1, 3, 4, 8, "f32", done=[1, 1, 0], end=1, change=lost)


@pytest.mark.parametrize("scale", [1e-3, 1.0, 80.0, 1e4, 1e30])
def test_sizes_of_logits(ctx, scale):
    _case(ctx, 2, 3, 4000, 6, "f32", spread=scale)
    _case(ctx, 2, 3, 4000, 6, "f32", change=lambda x, score: x.add_(scale * 100))
    if scale <= 1e4:
        _case(ctx, 2, 3, 4000, 6, "f32", change=lambda x, score: score.mul_(scale))


def test_signed_zeros_are_equal(ctx):
    def zeros(x, score):
        x.fill_(-1.0)
        x[:, 7], x[:, 5], x[:, 3] = 0.0, -0.0, -0.0

    _case(ctx, 1, 1, 3000, 3, "f32", change=zeros)


def test_in_place_and_without_ends(ctx):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(8, 700, generator=g)
    score = -torch.rand(8, generator=g)
    done = torch.tensor([0, 0, 1, 0, 0, 0, 0, 0], dtype=torch.uint8)
    want = _expect(x.numpy(), score.numpy(), 2, 4, 4, done.numpy(), 3)
    s, d, dev = score.cuda().view(2, 4), done.cuda().view(2, 4), x.cuda()
    token, parent = (torch.empty(2, 4, dtype=torch.int32, device="cuda") for _ in range(2))
    need = ctx.beam_select_workspace(2, 4, 700, 4)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    ctx.beam_select_device(vtq.F32, dev.data_ptr(), 700, 2, 4, 700, s.data_ptr(), 4, s.data_ptr(), token.data_ptr(),
                           parent.data_ptr(), ws.data_ptr(), need, stream(), done_ptr=d.data_ptr(), end_token=3,
                           out_done_ptr=d.data_ptr())
    torch.cuda.synchronize()
    _check((s, token, parent, d), want)
    before = token.clone()
    ctx.beam_select_device(vtq.F32, dev.data_ptr(), 700, 2, 4, 700, score.cuda().data_ptr(), 4, s.data_ptr(),
                           token.data_ptr(), parent.data_ptr(), ws.data_ptr(), need, stream())
    torch.cuda.synchronize()
    assert token.shape == before.shape


def test_streams_and_replayed_graphs(ctx):
    x = torch.randn(32, 30000, device="cuda").bfloat16()
    score = -torch.rand(32, device="cuda")
    want = _select(ctx, x, score, 8, 4, 8)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(_select(ctx, x, score, 8, 4, 8, wait=False))
    torch.cuda.synchronize()
    for got, _ in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, ws = _select(ctx, x, score, 8, 4, 8, wait=False)
    for _ in range(3):
        x.copy_(torch.randn(32, 30000, device="cuda"))
        score.uniform_(-3, 0)
        ws.fill_(255)
        eager = _select(ctx, x, score, 8, 4, 8)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


def test_more_rows_than_a_grid_takes(ctx):
    g = torch.Generator().manual_seed(1)
    rows, vocab = 70000, 33
    x = torch.randn(rows, vocab, generator=g)
    score = -torch.rand(rows, generator=g)
    token, parent = (t.cpu() for t in _select(ctx, x.cuda(), score.cuda(), rows // 2, 2, 2)[1:3])
    s = (torch.log_softmax(x.double(), -1) + score.double()[:, None]).view(rows // 2, -1)
    top = s.sort(dim=1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(token.long(), top % vocab)
    assert torch.equal(parent.long(), top // vocab + torch.arange(rows // 2)[:, None] * 2)


def test_logits_past_32_bits(ctx):
    rows, vocab = 9000, 1 << 19  # 2^32 and some elements, bf16
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    x[-1, -3], x[-2, 5], x[0, 9] = 20.0, 21.0, 22.0
    score = torch.full((rows,), -50.0, device="cuda")
    score[0] = score[-1] = score[-2] = 0.0
    outs = _select(ctx, x, score, 1 * rows // 3, 3, 1)
    token, parent = outs[1].cpu(), outs[2].cpu()
    assert (int(token[0]), int(parent[0])) == (9, 0) and (int(token[-1]), int(parent[-1])) == (5, rows - 2)
