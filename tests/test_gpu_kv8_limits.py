"""Attention over a paged 8-bit cache at the ends of f32's range."""
import pytest
import torch

from kv8 import Paged8
from test_gpu_kv8_attention import _attend

pytestmark = pytest.mark.gpu


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
