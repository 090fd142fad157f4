"""Plain 64-bit forms of the serving operators, and helpers of their tests."""
import math

import numpy as np
import torch

import vtq

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TAGS = {"f32": vtq.F32, "f16": vtq.F16, "bf16": vtq.BF16}
F32_HALF_STEP = 2.0 ** -24


def half_step(dtype):
    """A rounding is off by at most this much of the value."""
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """The step of subnormal values: a rounding there is off by at most half of it."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def up16(n):
    return (n + 15) // 16 * 16


def stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ int8

def quantize_exact(x):
    """(q, scale) of rows: the scale rounded once to f32, the quotient exact (64 bits hold it: two f32 numbers'
    quotient that is no half is further from one than 2^-53 of itself)."""
    x = x.double()
    top = x.abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0], dtype=torch.float64)
    scale = (top / 127.0).float()
    safe = torch.where((scale > 0) & torch.isfinite(scale), scale, torch.ones_like(scale)).double()
    q = torch.where(((scale > 0) & torch.isfinite(scale))[:, None], (x / safe[:, None]).round(), 0.0 * safe[:, None])
    return q.clamp(-127, 127).to(torch.int8), scale


# ------------------------------------------------------------------ rotation

def frequencies(rot, theta=10000.0, scaling=vtq.ROPE_SCALE_NONE, factor=1.0, original=0, low=0.0, high=0.0,
                factors=None):
    """Radians a position of every pair, and the magnitude."""
    out, magnitude = [], 1.0
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        if factors is not None:
            f /= float(np.float32(factors[i]))
        if scaling == vtq.ROPE_SCALE_LINEAR:
            f /= factor
        elif scaling == vtq.ROPE_SCALE_BANDS:
            lo, hi = low or 1.0, high or 4.0
            keep = min(1.0, max(0.0, (original * f / (2 * math.pi) - lo) / (hi - lo)))
            f = keep * f + (1 - keep) * f / factor
        elif scaling == vtq.ROPE_SCALE_YARN:
            lo, hi = low or 1.0, high or 32.0
            first = max(0, math.floor(rot * math.log(original / (hi * 2 * math.pi)) / (2 * math.log(theta))))
            last = min(rot - 1, math.ceil(rot * math.log(original / (lo * 2 * math.pi)) / (2 * math.log(theta))))
            ramp = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = (1 - ramp) * f + ramp * f / factor
            magnitude = 0.1 * math.log(factor) + 1.0
        out.append(f)
    return torch.tensor(out, dtype=torch.float64), magnitude


def rotate_exact(x, pos, freq, magnitude, layout):
    """x [tokens, heads, head_dim] turned to pos: (values, the sizes that their rounding errors go by)."""
    x = x.double().cpu()
    rot = 2 * freq.numel()
    angle = pos.double().cpu()[:, None] * freq[None, :]
    c, s = (torch.cos(angle) * magnitude)[:, None], (torch.sin(angle) * magnitude)[:, None]
    y, size = x.clone(), x.abs()
    ia = torch.arange(rot // 2) if layout == vtq.ROPE_HALF else torch.arange(0, rot, 2)
    ib = ia + (rot // 2 if layout == vtq.ROPE_HALF else 1)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia], size[..., ib] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return y, size, rot


def rotation_bound(y, size, dtype):
    """Cosine or sine, magnitude, product and sum each round once in f32 (4 half steps of the terms; the angle's own
    error, below 2^-52 of up to 2^20 turns, is a fifth), then the result rounds to its type."""
    return 5 * F32_HALF_STEP * size + half_step(dtype) * y.abs() * (1 + 1e-6) + smallest(dtype)


# ------------------------------------------------------------------ paged batches

class Paged:
    """A ragged batch over a paged cache whose pages are in no order.  layout "heads": pages x kv_heads x slots x
    head_dim; "slots": pages x slots x kv_heads x head_dim; "major": kv_heads x pages x slots x head_dim.  Slots that
    hold no token are NaN."""

    def __init__(self, q_lens, own_lens, prefix, kv_heads, head_dim, page, cache, seed=0, layout="heads", spare_pages=3,
                 extra_pages=0, device="cuda", fill=True):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.own_lens, self.prefix, self.page = list(q_lens), list(own_lens), prefix, page
        self.kv_heads, self.head_dim, self.cache_name, self.batch = kv_heads, head_dim, cache, len(q_lens)
        self.max_pages = max([1] + [-(-n // page) for n in own_lens]) + extra_pages
        n_prefix = -(-prefix // page)
        self.n_pages = n_prefix + self.batch * self.max_pages + spare_pages
        order = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        self.prefix_pages = order[:n_prefix].contiguous()
        self.pages = order[n_prefix:n_prefix + self.batch * self.max_pages].reshape(self.batch, self.max_pages).clone()
        self.q_start = torch.tensor([0] + list(np.cumsum(q_lens)), dtype=torch.int32)
        self.len = torch.tensor(own_lens, dtype=torch.int32)
        self.tokens = int(self.q_start[-1])
        shape = {"heads": (self.n_pages, kv_heads, page, head_dim), "slots": (self.n_pages, page, kv_heads, head_dim),
                 "major": (kv_heads, self.n_pages, page, head_dim)}[layout]
        self.layout = layout
        self.k = torch.full(shape, float("nan"), dtype=TYPES[cache])
        self.v = torch.full(shape, float("nan"), dtype=TYPES[cache])
        self.kh, self.vh = self.view(self.k), self.view(self.v)
        if fill:
            lists = [(self.prefix_pages, prefix)] + [(self.pages[b], n) for b, n in enumerate(own_lens)]
            for pages, n in lists:
                for t, view in ((0, self.kh), (1, self.vh)):
                    x = torch.randn(n, kv_heads, head_dim, generator=g).to(TYPES[cache])
                    for j0 in range(0, n, page):
                        m = min(page, n - j0)
                        view[int(pages[j0 // page]), :, :m] = x[j0:j0 + m].transpose(0, 1)
        if device == "cuda":
            self.to_device()

    def view(self, x):
        """A cache tensor as pages x kv_heads x slots x head_dim."""
        return {"heads": x, "slots": x.transpose(1, 2), "major": x.transpose(0, 1)}[self.layout]

    def to_device(self):
        self.dk, self.dv = self.k.cuda(), self.v.cuda()
        self.dlists = [t.cuda() for t in (self.q_start, self.len, self.pages, self.prefix_pages)]
        d = self.head_dim
        at = self.view(self.dk).stride()
        strides = dict(page_stride=at[0], head_stride=at[1], slot_stride=at[2])
        self.cache = vtq.KvCache(TAGS[self.cache_name], self.dk.data_ptr(), self.dv.data_ptr(), self.n_pages, self.page,
                                 self.kv_heads, d, **strides)
        self.desc = self.describe()

    def describe(self, max_q=None, max_len=0):
        return vtq.KvBatch(self.batch, self.dlists[0].data_ptr(), self.dlists[1].data_ptr(), self.dlists[2].data_ptr(),
                           self.max_pages, max_q=max(self.q_lens + [0]) if max_q is None else max_q, max_len=max_len,
                           prefix_len=self.prefix, prefix_pages=self.dlists[3].data_ptr() if self.prefix else None)

    def rows(self, view, pages, n):
        """n cached tokens in order: [kv_heads, n, head_dim] in 64 bits; pages outside the cache hold zeros."""
        out = torch.zeros(self.kv_heads, n, self.head_dim, dtype=torch.float64)
        for j0 in range(0, n, self.page):
            m, p = min(self.page, n - j0), int(pages[j0 // self.page])
            if 0 <= p < self.n_pages:
                out[:, j0:j0 + m] = view[p, :, :m].double()
        return out

    def places(self):
        """(sequence, place among its own tokens) of every token."""
        return [(b, self.own_lens[b] - n + i) for b, n in enumerate(self.q_lens) for i in range(n)]


def attention_exact(p, q, heads, scale):
    """(y, lse, bound of y, bound of lse) in 64 bits from the definition.  q [tokens, heads, head_dim] as stored.

    Bounds, u = 2^-24: a score's sum of head_dim products is off by at most (head_dim + 2) u of the sum of their
    magnitudes, the scaled score and its distance from the maximum by 4 u of the largest score, the exponential by
    4 u: together d.  Weights are then off by 2 d of themselves (their own error and the sum's), sums over n keys by
    n u; weights are rounded to 16 bits before the product where the queries are."""
    u, dtype = F32_HALF_STEP, q.dtype
    group = heads // p.kv_heads
    y = torch.zeros(p.tokens, heads, p.head_dim, dtype=torch.float64)
    lse = torch.full((p.tokens, heads), -math.inf, dtype=torch.float64)
    by, bl = torch.zeros_like(y), torch.zeros_like(lse)
    pk, pv = p.rows(p.kh, p.prefix_pages, p.prefix), p.rows(p.vh, p.prefix_pages, p.prefix)
    t = 0
    for b, n in enumerate(p.q_lens):
        if n == 0:
            continue
        m = max(0, min(p.own_lens[b], p.max_pages * p.page))
        ks = torch.cat([pk, p.rows(p.kh, p.pages[b], m)], 1)
        vs = torch.cat([pv, p.rows(p.vh, p.pages[b], m)], 1)
        for i in range(n):
            keys = p.prefix + max(0, min(m, p.own_lens[b] - n + i + 1))
            if keys:
                k, v = ks[:, :keys], vs[:, :keys]
                qt = q[t].double().cpu().view(p.kv_heads, group, -1)
                s = torch.matmul(qt, k.transpose(1, 2)) * scale
                mag = (torch.matmul(qt.abs(), k.abs().transpose(1, 2)) * scale).amax(-1)
                d = (p.head_dim + 2) * u * mag + 4 * u * s.abs().amax(-1) + 4 * u
                w = torch.softmax(s, -1)
                out, size = torch.matmul(w, v), torch.matmul(w, v.abs())
                rel = 2.1 * d + keys * u + (0 if dtype == torch.float32 else half_step(dtype) * 1.01)
                y[t], lse[t] = out.view(heads, -1), torch.logsumexp(s, -1).view(-1)
                by[t] = (rel[..., None] * size + half_step(dtype) * out.abs() * 1.01 + smallest(dtype)
                         + (0 if dtype == torch.float32 else smallest(dtype) * v.abs().amax() * keys)).view(heads, -1)
                bl[t] = (d + keys * u).view(-1) + 4 * u * lse[t].abs()
            t += 1
    return y, lse, by, bl


def within(got, want, bound, what):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= bound) & ~((got == want) | (got.isnan() & want.isnan()))
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: got {float(got[i])}, "
                             f"want {float(want[i])}, allowed {float(bound[i])}")
