"""int8 activations and the int8 product (vtq_quantize_i8_device, vtq_linear_i8_device) against 64 bits."""
import pytest
import torch

import vtq
from serving import F32_HALF_STEP, TAGS, TYPES, half_step, quantize_exact, smallest, stream, up16, within

pytestmark = pytest.mark.gpu


def _quantize(ctx, x, ld_q=None):
    rows, n = x.shape
    ld_q = up16(n) if ld_q is None else ld_q
    q = torch.full((rows, ld_q), 99, dtype=torch.int8, device="cuda")
    s = torch.full((rows,), float("nan"), device="cuda")
    name = next(k for k, t in TYPES.items() if t == x.dtype)
    ctx.quantize_i8_device(TAGS[name], x.data_ptr(), x.stride(0), q.data_ptr(), ld_q, s.data_ptr(), rows, n, stream())
    torch.cuda.synchronize()
    return q, s


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 4096), (3, 15), (2, 17), (5, 100), (1, 4097), (7, 2048), (2, 11008),
                                    (1, 14336), (1, 20000), (1, 131071), (300, 777), (70000, 32)])
def test_quantize_equals_the_definition(ctx, dtype, rows, n):
    g = torch.Generator().manual_seed(rows * 1000 + n)
    x = torch.randn(rows, n, generator=g).to(TYPES[dtype])
    q, s = _quantize(ctx, x.cuda())
    want_q, want_s = quantize_exact(x)
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q[:, :n].cpu(), want_q)
    assert not q[:, n:].any()


def test_quantize_halves_go_to_even_and_borders_hold(ctx):
    # scale 1: the halves themselves; a scale of 3 steps: quotients next to halves
    a = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5, 0.0, -0.0]])
    s = float(torch.tensor(1.1).float())
    k = torch.arange(-126, 127).double()
    b = torch.cat([torch.tensor([127 * s]).double(), (k + 0.5) * s]).float()[None]
    near = torch.cat([b, torch.nextafter(b, torch.full_like(b, 9e9)), torch.nextafter(b, torch.full_like(b, -9e9))], 1)
    for x in (a, b, near, near * 2.0 ** -100, near * 2.0 ** 100):
        q, sc = _quantize(ctx, x.cuda())
        want_q, want_s = quantize_exact(x)
        assert torch.equal(sc.cpu(), want_s)
        assert torch.equal(q[:, :x.shape[1]].cpu(), want_q)


def test_quantize_zero_subnormal_and_not_finite_rows(ctx):
    tiny = 2.0 ** -149
    x = torch.zeros(6, 40)
    x[1, 3] = 200 * tiny  # scale 2 steps: the quotient 100
    x[2, 3] = 63 * tiny   # scale 0
    x[3, 3], x[3, 4] = 190 * tiny, 5 * tiny  # scale 1 step: 190 is cut to 127
    x[4, 5], x[4, 6] = float("inf"), 3.0
    x[5, 5], x[5, 6], x[5, 7] = float("nan"), float("inf"), 3.0
    q, s = _quantize(ctx, x.cuda())
    assert s[:4].tolist() == [0.0, 2 * tiny, 0.0, tiny]
    assert q[1, 3] == 100 and q[3, 3] == 127 and q[3, 4] == 5 and not q[0].any() and not q[2].any()
    assert s[4].item() == float("inf") and s[5].isnan() and not q[4:].any()


def test_quantize_strided_unaligned_rows(ctx):
    g = torch.Generator().manual_seed(5)
    for dtype in ("bf16", "f32"):
        wide = torch.randn(6, 1001, generator=g).to(TYPES[dtype])
        x = wide.cuda()[:, 3:3 + 517]
        q, s = _quantize(ctx, x, ld_q=640)
        want_q, want_s = quantize_exact(wide[:, 3:520])
        assert torch.equal(s.cpu(), want_s) and torch.equal(q[:, :517].cpu(), want_q) and not q[:, 517:].any()


def _product(ctx, m, k, n, out, bias, seed, garbage=True, ld_y=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = up16(k)
    xq = torch.zeros(m, ld, dtype=torch.int8, device="cuda")
    xq[:, :k] = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    wq = torch.full((n, ld), 113 if garbage else 0, dtype=torch.int8, device="cuda")  # anything past the row
    wq[:, :k] = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    xs = torch.rand(m, generator=g, device="cuda") * 0.01 + 1e-4
    ws = torch.rand(n, generator=g, device="cuda") * 0.01 + 1e-4
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    ld_y = n if ld_y is None else ld_y
    y = torch.full((m, ld_y), 7.0, dtype=TYPES[out], device="cuda")
    ctx.linear_i8_device(xq.data_ptr(), ld, xs.data_ptr(), wq.data_ptr(), ld, ws.data_ptr(),
                         None if b is None else b.data_ptr(), TAGS[out], y.data_ptr(), ld_y, m, k, n, stream())
    torch.cuda.synchronize()
    acc = xq[:, :k].double() @ wq[:, :k].double().t().contiguous()  # whole numbers below 2^53: exact
    prod = acc * xs.double()[:, None] * ws.double()[None, :]
    want = prod + (b.double() if bias else 0.0)
    # the sum rounds to f32, then two products and the bias: four half steps; then to the type
    bound = 4.01 * F32_HALF_STEP * (prod.abs() + (b.double().abs() if bias else 0.0)) \
        + half_step(TYPES[out]) * want.abs() * (1 + 1e-6) + smallest(TYPES[out])
    within(y[:, :n], want.cpu(), bound.cpu(), f"{m}x{k}->{n} {out}")
    assert (y[:, n:] == 7.0).all()
    return y


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 16, 16), (1, 4096, 4096), (2, 100, 33), (3, 256, 1000), (16, 2048, 5632),
                                   (17, 4096, 256), (19, 11008, 512), (33, 1001, 777), (64, 4096, 4096), (65, 640, 129),
                                   (100, 5000, 2000), (128, 14336, 300), (200, 64, 4100), (255, 4112, 257),
                                   (512, 4096, 1000), (700, 130, 2049), (1025, 896, 4864),
                                   (190, 4100, 11001), (250, 11000, 4090), (1001, 4112, 11003)])
def test_product(ctx, m, k, n, out):
    _product(ctx, m, k, n, out, bias=(m + n) % 2 == 0, seed=m * 7 + k * 3 + n)


def test_product_over_more_channels_and_tokens_than_a_launch(ctx):
    _product(ctx, 1, 40, (1 << 20) + 300, "bf16", True, 11)
    _product(ctx, 70, 33, (1 << 20) + 17, "f32", False, 12)
    _product(ctx, 1048560 + 100, 16, 19, "f16", True, 13)


def test_product_at_the_largest_sums(ctx):
    # 131071 products of 127 * -128: the sum is within 32 bits
    k, ld = 131071, up16(131071)
    for m in (1, 40, 300):
        xq = torch.zeros(m, ld, dtype=torch.int8, device="cuda")
        xq[:, :k] = 127
        wq = torch.full((48, ld), -128, dtype=torch.int8, device="cuda")
        one = torch.ones(max(m, 48), device="cuda")
        y = torch.zeros(m, 48, device="cuda")
        ctx.linear_i8_device(xq.data_ptr(), ld, one.data_ptr(), wq.data_ptr(), ld, one.data_ptr(), None, vtq.F32,
                             y.data_ptr(), 48, m, k, 48, stream())
        assert (y == float(torch.tensor(-127.0 * 128 * k, dtype=torch.float32))).all()


def test_product_of_no_inputs_is_the_bias(ctx):
    b = torch.arange(20, dtype=torch.float32, device="cuda")
    y = torch.full((3, 20), 7.0, device="cuda")
    ctx.linear_i8_device(None, 0, None, None, 0, None, b.data_ptr(), vtq.F32, y.data_ptr(), 20, 3, 0, 20, stream())
    assert (y == b).all()
    ctx.linear_i8_device(None, 0, None, None, 0, None, None, vtq.F32, y.data_ptr(), 20, 3, 0, 20, stream())
    assert not y.any()


def test_product_into_part_of_wider_rows(ctx):
    for m in (2, 90, 600):
        _product(ctx, m, 320, 500, "bf16", True, 3, ld_y=777)


def test_rows_that_are_not_finite_give_nan(ctx):
    for m in (4, 200):
        x = torch.randn(m, 512, device="cuda")
        x[1, 100], x[2, 7] = float("inf"), float("nan")
        q, s = _quantize(ctx, x)
        w = torch.ones(64, 512, dtype=torch.int8, device="cuda")
        ws = torch.ones(64, device="cuda")
        y = torch.zeros(m, 64, device="cuda")
        ctx.linear_i8_device(q.data_ptr(), 512, s.data_ptr(), w.data_ptr(), 512, ws.data_ptr(), None, vtq.F32,
                             y.data_ptr(), 64, m, 512, 64, stream())
        assert y[1:3].isnan().all() and y[0].isfinite().all() and y[3:].isfinite().all()


def test_product_past_two_gigabytes_of_outputs_and_weights(ctx):
    # 600 x 2^22 bytes of weights and outputs past 2^31 elements: offsets in 64 bits
    n, k, m = 1 << 22, 512, 600
    w = torch.ones(n, k, dtype=torch.int8, device="cuda")
    w[-1] = 3
    x = torch.full((m, k), 2, dtype=torch.int8, device="cuda")
    x[-1] = -1
    one = torch.ones(n, device="cuda")
    y = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    ctx.linear_i8_device(x.data_ptr(), k, one.data_ptr(), w.data_ptr(), k, one.data_ptr(), None, vtq.BF16, y.data_ptr(),
                         n, m, k, n, stream())
    assert (y[:-1, :-1] == 1024).all() and (y[:-1, -1] == 6 * k).all()
    assert (y[-1, :-1] == -512).all() and y[-1, -1] == -1536


@pytest.mark.parametrize("m", [1, 20, 300])
def test_captured_products_replay(ctx, m):
    k, n = 1024, 512
    x = torch.randn(m, k, device="cuda")
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda")
    ws = torch.rand(n, device="cuda")

    def step(y, q, s):
        ctx.quantize_i8_device(vtq.F32, x.data_ptr(), k, q.data_ptr(), k, s.data_ptr(), m, k, stream())
        ctx.linear_i8_device(q.data_ptr(), k, s.data_ptr(), w.data_ptr(), k, ws.data_ptr(), None, vtq.F32, y.data_ptr(),
                             n, m, k, n, stream())

    bufs = [(torch.zeros(m, n, device="cuda"), torch.zeros(m, k, dtype=torch.int8, device="cuda"),
             torch.zeros(m, device="cuda")) for _ in range(2)]
    step(*bufs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*bufs[1])
    for i in range(3):
        x.copy_(torch.randn(m, k, device="cuda") * (i + 1))
        step(*bufs[0])
        bufs[1][0].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bufs[0][0], bufs[1][0])
