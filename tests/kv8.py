"""Plain 64-bit forms of the operators over 8-bit caches, and helpers of their tests."""
import math

import numpy as np
import torch

import vtq
from serving import F32_HALF_STEP, TAGS, Paged, half_step, smallest

LEAST, MOST = -117, 119  # exponents of scales
E4M3_HALF_STEP = 2.0 ** -4
E4M3_SMALLEST = 2.0 ** -9
# weights are sums of one, two or three bf16 parts
WEIGHT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -24}
PARTS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}


def exponent_for(top):
    """The least e with top <= 448 * 2^e, from the definition (top a Python float)."""
    e = LEAST
    while e < MOST and top > 448.0 * 2.0 ** e:
        e += 1
    return e


def exponents(byte):
    return byte.to(torch.int64).clamp(127 + LEAST, 127 + MOST) - 127


def quantize(x, e):
    """x (f32) over 2^e as e4m3 codes: to the nearest, 448 at most, infinities and NaN to NaN."""
    y = torch.ldexp(x.double(), -torch.as_tensor(e)).clamp(-448.0, 448.0)
    y = torch.where(torch.isfinite(x), y, math.nan)
    return y.float().to(torch.float8_e4m3fn).view(torch.uint8)  # (a quotient by 2^e is an f32 number, or below e4m3's least)


def values(codes, byte, block):
    """What codes [pages, heads, slots, d] under scale bytes [pages, heads, slots / block] stand for, in 64 bits."""
    e = exponents(byte).repeat_interleave(block, -1)[..., None]
    return torch.ldexp(codes.view(torch.float8_e4m3fn).double(), e)


class Paged8(Paged):
    """A ragged batch over a paged 8-bit cache.  Layouts as Paged; slots that hold no token are NaN, blocks that hold
    none have any scale."""

    def __init__(self, q_lens, own_lens, prefix, kv_heads, head_dim, page, block=16, seed=0, layout="heads",
                 spare_pages=3, extra_pages=0, device="cuda", fill=True, loud=1.0):
        super().__init__(q_lens, own_lens, prefix, kv_heads, head_dim, page, "f32", seed=seed, layout=layout,
                         spare_pages=spare_pages, extra_pages=extra_pages, device=None, fill=False)
        self.block = block
        g = torch.Generator().manual_seed(seed + 77)
        self.kc = torch.full(self.k.shape, 0x7F, dtype=torch.uint8)
        self.vc = self.kc.clone()
        scales = (kv_heads, self.n_pages, page // block) if layout == "major" else (self.n_pages, kv_heads, page // block)
        self.ks, self.vs = (torch.randint(0, 256, scales, generator=g, dtype=torch.uint8) for _ in range(2))
        self.k = self.v = None
        if fill:
            lists = [(self.prefix_pages, prefix)] + [(self.pages[b], n) for b, n in enumerate(own_lens)]
            for pages, n in lists:
                for j0 in range(0, n, block):
                    m, p = min(block, n - j0), int(pages[j0 // page])
                    s = slice(j0 % page, j0 % page + m)
                    for codes, scale in ((self.kc, self.ks), (self.vc, self.vs)):
                        x = torch.randn(kv_heads, m, head_dim, generator=g)
                        x *= loud * torch.exp2(0.7 * torch.randn(kv_heads, 1, 1, generator=g))
                        for h in range(kv_heads):
                            e = exponent_for(float(x[h].abs().amax()))
                            self.view(codes)[p, h, s] = quantize(x[h], e)
                            self.scale_view(scale)[p, h, j0 % page // block] = e + 127
        self.refresh()
        if device == "cuda":
            self.to_device()

    def scale_view(self, x):
        return x.transpose(0, 1) if self.layout == "major" else x

    def refresh(self):
        """kh and vh, pages x kv_heads x slots x head_dim, from codes and scales."""
        self.kh = values(self.view(self.kc).contiguous(), self.scale_view(self.ks), self.block)
        self.vh = values(self.view(self.vc).contiguous(), self.scale_view(self.vs), self.block)

    def from_device(self):
        self.kc, self.vc, self.ks, self.vs = (t.cpu() for t in (self.dk, self.dv, self.dks, self.dvs))
        self.refresh()

    def to_device(self):
        self.dk, self.dv, self.dks, self.dvs = (t.cuda() for t in (self.kc, self.vc, self.ks, self.vs))
        self.dlists = [t.cuda() for t in (self.q_start, self.len, self.pages, self.prefix_pages)]
        at, scale = self.view(self.dk).stride(), self.scale_view(self.dks).stride()
        self.cache = vtq.Kv8Cache(self.dk.data_ptr(), self.dv.data_ptr(), self.dks.data_ptr(), self.dvs.data_ptr(),
                                  self.n_pages, self.page, self.kv_heads, self.head_dim, block=self.block,
                                  page_stride=at[0], head_stride=at[1], slot_stride=at[2], scale_page_stride=scale[0],
                                  scale_head_stride=scale[1])
        self.desc = self.describe()


def attention8_exact(p, q, heads, scale):
    """(y, lse, bound of y, bound of lse) in 64 bits from the definition.

    Bounds, u = 2^-24, as for the wider caches: a score is a sum of head_dim products a part, off by at most
    (parts head_dim + 2) u of the sum of their magnitudes, its distance from the maximum by 4 u of the largest score,
    the exponential by 4 u: together d.  Weights are off by 2 d of themselves, sums over n keys and parts by parts n u;
    weights are rounded to their parts before the product.  Parts below 2^-126 may be lost: that of a query times
    any key, that of a weight times any value."""
    u, dtype, parts = F32_HALF_STEP, q.dtype, PARTS[q.dtype]
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
                lost = 2.0 ** -126 * scale * p.head_dim * k.abs().amax((1, 2))[:, None]
                d = (parts * p.head_dim + 2) * u * mag + 4 * u * s.abs().amax(-1) + 4 * u + lost
                w = torch.softmax(s, -1)
                out, size = torch.matmul(w, v), torch.matmul(w, v.abs())
                rel = 2.1 * d + parts * keys * u + WEIGHT[dtype] * 1.01
                y[t], lse[t] = out.view(heads, -1), torch.logsumexp(s, -1).view(-1)
                by[t] = (rel[..., None] * size + half_step(dtype) * out.abs() * 1.01 + smallest(dtype)
                         + 2.0 ** -126 * v.abs().amax() * keys).view(heads, -1)
                bl[t] = (d + keys * u).view(-1) + 4 * u * lse[t].abs()
            t += 1
    return y, lse, by, bl


def append8_exact(p, which, x, size):
    """Checks the cache on the device against p's state before the call (p.kc, p.ks, ... still hold it).  x: the
    rotated keys or the values in 64 bits, [tokens, kv_heads, head_dim]; size: how far the kernel's f32 x may be off
    each.  Every block, element and scale: those of the call's tokens by the definition, all others bit for bit."""
    before = p.view(p.kc if which == "k" else p.vc).contiguous()
    scale = p.scale_view(p.ks if which == "k" else p.vs).contiguous()
    got = p.view((p.dk if which == "k" else p.dv).cpu()).contiguous()
    got_scale = p.scale_view((p.dks if which == "k" else p.dvs).cpu()).contiguous()
    want, want_scale = before.clone(), scale.clone()
    blocks = {}
    for t, (b, place) in enumerate(p.places()):
        if place < 0 or place // p.page >= p.max_pages or not 0 <= int(p.pages[b, place // p.page]) < p.n_pages:
            continue
        blocks.setdefault((int(p.pages[b, place // p.page]), place % p.page // p.block), []).append((place % p.page, t))
    for (page, i), tokens in blocks.items():
        slots, ts = [s for s, _ in tokens], [t for _, t in tokens]
        first = min(slots) - i * p.block
        for h in range(p.kv_heads):
            v, off = x[ts, h], size[ts, h]
            finite = torch.isfinite(v)
            top = float(torch.where(finite, v.abs(), 0.0).amax())
            slack = float(torch.where(finite, off, 0.0).amax())
            allowed = {exponent_for(top - slack), exponent_for(top), exponent_for(top + slack)}
            old = int(exponents(scale[page, h, i]))
            if first > 0:
                allowed = {max(e, old) for e in allowed}
            e = int(got_scale[page, h, i]) - 127
            assert e in allowed, (which, page, i, h, e, allowed)
            want_scale[page, h, i] = e + 127
            if first > 0 and e > old:
                s = slice(i * p.block, i * p.block + first)
                turned = torch.ldexp(before[page, h, s].view(torch.float8_e4m3fn).float(), torch.tensor(old - e))
                assert same_codes(got[page, h, s], turned.to(torch.float8_e4m3fn).view(torch.uint8)), (which, page, i, h)
                want[page, h, s] = got[page, h, s]
            stored = torch.ldexp(got[page, h, slots].view(torch.float8_e4m3fn).double(), torch.tensor(e))
            bound = (off + E4M3_HALF_STEP * v.abs() * (1 + 1e-6) + 0.5 * E4M3_SMALLEST * 2.0 ** e)
            bad = torch.where(finite, (stored - v).abs() > bound, ~stored.isnan())
            assert not bad.any(), (which, page, i, h, stored[bad][:3], v[bad][:3])
            if slack == 0:
                assert same_codes(got[page, h, slots], quantize(v.float(), e)), (which, page, i, h)
            want[page, h, slots] = got[page, h, slots]
    assert torch.equal(got, want) and torch.equal(got_scale, want_scale), which


def same_codes(a, b):
    nan = ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)
    return bool(((a == b) | nan).all())


def log_softmax(x):
    """In 64 bits with numpy, a row at a time."""
    x = np.asarray(x, dtype=np.float64)
    top = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        return x - (top + np.log(np.exp(x - top).sum(-1, keepdims=True)))


__all__ = ["Paged8", "TAGS", "append8_exact", "attention8_exact", "exponent_for", "exponents", "log_softmax", "quantize",
           "same_codes", "values"]
