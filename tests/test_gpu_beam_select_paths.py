"""Choosing the best continuations of beams where a group's lists are more than its join holds in registers, without
ends, and of rows whose sums are equal or nearly so."""
import numpy as np
import pytest
import torch

import vtq
from kv8 import log_softmax
from serving import stream
from test_gpu_beam_select import INF, NAN, _case, _check, _expect, _select

pytestmark = pytest.mark.gpu

# A join holds 4096 entries at most: beams x parts of a row (of 2048 logits, or 8192 where rows are many) x n_out.
LARGE = [(1, 8, 128000, 16), (2, 8, 128256, 16), (1, 16, 32000, 32), (1, 64, 4100, 64), (10, 64, 9000, 64), (1, 3, 250000, 33)]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab,n_out", LARGE)
def test_more_lists_than_a_join_holds(ctx, name, groups, beams, vocab, n_out):
    _case(ctx, groups, beams, vocab, n_out, name, seed=vocab)


@pytest.mark.parametrize("groups,beams,vocab,n_out", [(1, 8, 128000, 16), (1, 64, 4100, 64), (10, 64, 9000, 64)])
def test_alike_masked_and_ended_rows_of_many_lists(ctx, groups, beams, vocab, n_out):
    rows = groups * beams

    def same(x, score):
        x.fill_(0.5)
        score.fill_(-2.0)

    def one_in_each(x, score):  # as many equal candidates as lists
        x.fill_(-3.0)
        x[:, ::2048] = 1.0
        score.fill_(-1.0)

    def first(x, score):
        x.copy_(x[0].expand_as(x).clone())
        score.fill_(-INF)
        score[::beams] = 0.0

    def masked(x, score):
        y = torch.full_like(x, -INF)
        y[:, 5:vocab:vocab // 3] = x[:, 5:vocab:vocab // 3]
        x.copy_(y)

    def bad(x, score):
        x[0, 5], x[1, vocab - 1], x[2, :] = NAN, INF, -INF
        score[3], score[4] = NAN, -INF

    def none(x, score):
        x[:, 0] = NAN

    for change in (same, one_in_each, first, masked, bad, none):
        _case(ctx, groups, beams, vocab, n_out, "f32", change=change)
    g = torch.Generator().manual_seed(5)
    done = (torch.rand(rows, generator=g) < 0.4).to(torch.uint8).tolist()
    _case(ctx, groups, beams, vocab, n_out, "f32", done=done, end=2)
    done = [1] * rows
    done[rows // 2] = 0
    _case(ctx, groups, beams, vocab, n_out, "f32", done=done, end=-1)


@pytest.mark.parametrize("groups,beams,vocab,n_out", [(2, 4, 700, 4), (3, 5, 9000, 8), (1, 8, 128000, 16)])
def test_without_ends(ctx, groups, beams, vocab, n_out):
    g = torch.Generator().manual_seed(vocab)
    x = 3 * torch.randn(groups * beams, vocab, generator=g)
    score = -torch.rand(groups * beams, generator=g)
    dx, ds = x.cuda(), score.cuda()
    out_score = torch.full((groups, n_out), 7.0, device="cuda")
    token, parent = (torch.full((groups, n_out), 7, dtype=torch.int32, device="cuda") for _ in range(2))
    need = ctx.beam_select_workspace(groups, beams, vocab, n_out)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    for end in (-1, 3):  # with an end, but nobody who asks who ended
        ctx.beam_select_device(vtq.F32, dx.data_ptr(), vocab, groups, beams, vocab, ds.data_ptr(), n_out,
                               out_score.data_ptr(), token.data_ptr(), parent.data_ptr(), ws.data_ptr(), need, stream(),
                               end_token=end)
        torch.cuda.synchronize()
        want = _expect(x.numpy(), score.numpy(), groups, beams, n_out)
        _check((out_score, token, parent, torch.zeros_like(token)), want)
        assert (ws[need:] == 255).all()
        out_score.fill_(7.0), token.fill_(7), parent.fill_(7)


@pytest.mark.parametrize("vocab,n_out", [(64, 12), (3000, 30), (20000, 64), (130000, 20)])
def test_rows_that_are_equal_but_for_their_order_or_a_constant(ctx, vocab, n_out):
    # a row, the same permuted, the same shifted by a constant (exact in f32), and the same again: equal sums in exact
    # arithmetic.  Sums are right to 2^-32, so that those of two rows may differ by 2^-31 and come in either order; within a
    # row, and between rows of the same logits, the order is that of the definition.
    g = torch.Generator().manual_seed(vocab)
    row = torch.round(2.5 * torch.randn(vocab, generator=g) * 2 ** 10) / 2 ** 10
    perm = torch.randperm(vocab, generator=g)
    x = torch.stack([row, row[perm], row + 8.0, row])
    score = torch.full((4,), -1.25)
    outs = _select(ctx, x.cuda(), score.cuda(), 1, 4, n_out)
    got = [(int(p), int(t)) for p, t in zip(outs[2].cpu()[0], outs[1].cpu()[0])]
    assert len(set(got)) == n_out
    exact = -1.25 + log_softmax(x.double().numpy())
    best = np.sort(exact.reshape(-1))[::-1][:n_out]
    for (p, t), want, s in zip(got, best, outs[0].cpu()[0].tolist()):
        assert abs(exact[p, t] - want) <= 2.0 ** -31 and abs(s - want) <= 2.0 ** -24 * abs(want) * 1.001 + 2.0 ** -31
    for r in range(4):
        of_row = [t for p, t in got if p == r]
        assert of_row == sorted(of_row, key=lambda t: (-float(x[r, t]), t))
    for t in {t for _, t in got}:  # the first and the last row tie exactly: a token of the last follows the first's
        if (3, t) in got:
            assert (0, t) in got and got.index((0, t)) < got.index((3, t))
