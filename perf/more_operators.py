"""Performance cases of decoding with beams over an 8-bit cache: append and attention where keys and values are e4m3
with a scale a block of tokens and head, selection over beams and vocabulary, and the cache's pages (forked, freed,
grown, compacted, copied).

A case is one of
  append     a step's keys (rotated) and values of a ragged batch into an 8-bit paged cache, its queries rotated;
  attention  a ragged batch against a prefix that all sequences share and the pages of their own, in 8 bits;
  beam       the best continuations of groups of beams over their vocabulary;
  reorder    the page tables of the next batch from the sequences that it continues, and the copies that this takes;
  compact    the pages in use moved to the low end of the cache, in tables and on every layer.

`run` computes a case in elementary torch operations, or, where `own` is set, through the library.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_LEAST, _MOST = -117, 119  # exponents of scales


def _append(batch, q_max, prefix, own_max, heads, kv_heads, head_dim, rot_dim, layout, page, block, dtype, ragged):
    return {"kind": "append", "batch": batch, "q_max": q_max, "prefix": prefix, "own_max": own_max, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "rot_dim": rot_dim, "layout": layout, "page": page,
            "block": block, "dtype": dtype, "ragged": ragged}


def _attention(batch, q_max, prefix, own_max, heads, kv_heads, head_dim, page, block, dtype, ragged):
    return {"kind": "attention", "batch": batch, "q_max": q_max, "prefix": prefix, "own_max": own_max, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "block": block, "dtype": dtype, "ragged": ragged}


def _beam(groups, beams, vocab, keep, dtype, done):
    return {"kind": "beam", "groups": groups, "beams": beams, "vocab": vocab, "keep": keep, "dtype": dtype,
            "done": done}


def _pages(kind, batch, max_pages, page, n_pages, layers, kv_heads, head_dim, cache, parents="", grow=1, live=1.0):
    return {"kind": kind, "batch": batch, "max_pages": max_pages, "page": page, "n_pages": n_pages, "layers": layers,
            "kv_heads": kv_heads, "head_dim": head_dim, "cache": cache, "parents": parents, "grow": grow, "live": live}


def listed():
    return [
        # 32 sequences, one new token each, behind a shared system prompt
        {"name": "append_decode32", **_append(32, 1, 2048, 700, 32, 8, 128, 128, "half", 16, 16, "bf16", 21)},
        # packed prompts of five sequences, part of each head rotated, f32 activations
        {"name": "append_prompts", **_append(5, 1200, 0, 1200, 32, 8, 80, 32, "interleaved", 64, 32, "f32", 22)},
        # four sequences of the 1.1B model in f32
        {"name": "attention_decode4_f32", **_attention(4, 1, 500, 90, 32, 4, 64, 16, 16, "f32", 23)},
        # drafts of up to six tokens to be checked at once, odd lengths, a short prefix
        {"name": "attention_drafts16", **_attention(16, 6, 1003, 4000, 24, 8, 96, 32, 16, "f16", 24)},
        # 64 chats behind a system prompt of 8192 tokens
        {"name": "attention_batch64_8k", **_attention(64, 1, 8192, 512, 32, 8, 128, 16, 16, "bf16", 25)},
        # 128 questions about one document
        {"name": "attention_batch128_32k", **_attention(128, 1, 32768, 1024, 32, 8, 128, 64, 32, "bf16", 26)},
        # four beams of the 1.1B model, f32 logits as its linear gives them
        {"name": "beam_1x4_32000", **_beam(1, 4, 32000, 8, "f32", 0)},
        # 64 requests of eight beams, a large vocabulary, some beams ended
        {"name": "beam_64x8_128000", **_beam(64, 8, 128000, 16, "bf16", 60)},
        # eight requests of four beams after a selection, the 1.1B model's 22 layers
        {"name": "reorder_beams32", **_pages("reorder", 32, 64, 16, 1400, 22, 4, 64, "bf16", "beams", 1)},
        # 256 sequences on a large 8-bit cache: some end, some fork, all may grow by a draft
        {"name": "reorder_mixed256", **_pages("reorder", 256, 256, 16, 40000, 4, 8, 128, "e4m3", "mixed", 6)},
        # a half-empty cache of the 1.1B model closed up
        {"name": "compact_1000", **_pages("compact", 24, 40, 16, 1000, 22, 4, 64, "f16", live=0.6)},
        # a large 8-bit cache after many requests have ended
        {"name": "compact_4096", **_pages("compact", 64, 80, 32, 4096, 8, 8, 128, "e4m3", live=0.55)},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One more case: any of the kinds, their types and layouts, sizes over the listed ranges."""
    kind = rng.choice(["append", "attention", "attention", "beam", "beam", "reorder", "compact"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "beam":
        while True:
            groups, beams = _log_int(rng, 1, 64), _log_int(rng, 1, 16)
            vocab = _log_int(rng, 1000, 256000)
            if groups * beams * vocab <= 64 * 8 * 128000:
                done = rng.randint(0, groups * beams // 8) if rng.random() < 0.5 else 0
                return _beam(groups, beams, vocab, beams * rng.choice([1, 2, 2]), dtype, done)
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind in ("reorder", "compact"):
        cache = rng.choice(["e4m3", "e4m3", "bf16", "f16", "f32"])
        size = {"e4m3": 1, "bf16": 2, "f16": 2, "f32": 4}[cache]
        while True:
            batch, max_pages = _log_int(rng, 4, 256), _log_int(rng, 8, 256)
            layers = _log_int(rng, 1, 32)
            n_pages = int(batch * max_pages * (0.6 + 0.5 * rng.random())) + 40
            if n_pages * layers * kv_heads * page * head_dim * size <= 1 << 30:
                return _pages(kind, batch, max_pages, page, n_pages, layers, kv_heads, head_dim, cache,
                              rng.choice(["beams", "mixed"]), _log_int(rng, 1, 40), 0.3 + 0.5 * rng.random())
    group = rng.choice([1, 2, 4, 4, 7, 8])
    heads = kv_heads * group
    block = rng.choice([b for b in (16, 16, 32, 64) if b <= page])
    ragged = rng.randint(100, 10 ** 6)
    if kind == "append":
        q_max = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1200)
        batch = max(1, min(_log_int(rng, 1, 128), 5000 // q_max))
        return _append(batch, q_max, _log_int(rng, 1, 32768), q_max + _log_int(rng, 1, 2000), heads, kv_heads, head_dim,
                       rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4]),
                       rng.choice(["interleaved", "half"]), page, block, dtype, ragged)
    while True:
        q_max = 1 if rng.random() < 0.5 else _log_int(rng, 2, 300)
        batch = _log_int(rng, 1, 128)
        prefix = 0 if rng.random() < 0.15 else _log_int(rng, 16, 32768)
        own_max = q_max + _log_int(rng, 1, 4000)
        rows = batch * q_max * heads
        most = 128 * 32 * (32768 + 1024) * 128 // {"bf16": 1, "f16": 2, "f32": 4}[dtype]  # products a weight
        if rows * (prefix + own_max) * head_dim <= most and batch * own_max * kv_heads * head_dim <= 1 << 27:
            return _attention(batch, q_max, prefix, own_max, heads, kv_heads, head_dim, page, block, dtype, ragged)


# ------------------------------------------------------------------ lengths, angles, scales

def _lengths(case):
    """New tokens and cached own tokens (the new ones among them) of every sequence."""
    rng = random.Random(case["ragged"])
    q = [rng.randint((case["q_max"] + 1) // 2, case["q_max"]) for _ in range(case["batch"])]
    q[0] = case["q_max"]
    kv = [n + rng.randint((case["own_max"] - case["q_max"]) // 2, case["own_max"] - case["q_max"]) for n in q]
    return q, kv


def _rotate(case, x, pos):
    """x [tokens, heads, head_dim] at pos, in 32 bits; the angles in 64."""
    r = case["rot_dim"]
    i = torch.arange(r // 2, dtype=torch.float64, device=x.device)
    angles = pos.double()[:, None] * torch.exp(-2.0 * i / r * math.log(10000.0))[None, :]
    c, s = torch.cos(angles).float()[:, None, :], torch.sin(angles).float()[:, None, :]
    x = x.float()
    out = x.clone()
    if case["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        out[..., : r // 2], out[..., r // 2: r] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2], out[..., 1:r:2] = a * c - b * s, b * c + a * s
    return out


def _exponent(top):
    """The least e with top <= 448 * 2^e."""
    m, e = torch.frexp(top)  # top = m * 2^e, 1/2 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(top > 0, e, _LEAST).clamp(_LEAST, _MOST)


def _to_e4m3(x, e):
    y = torch.ldexp(x, -e)
    return torch.where(torch.isfinite(x), y.clamp(-448.0, 448.0), math.nan).to(torch.float8_e4m3fn)


# ------------------------------------------------------------------ inputs

_context = None


def _ctx():
    """The program's one context."""
    global _context
    if _context is None:
        import os
        import sys

        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vitni-tensor_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import vtq

        _context = vtq.Context(0)
    return _context


def _tag(name):
    import vtq

    return {"f32": vtq.F32, "f16": vtq.F16, "bf16": vtq.BF16}[name]


def _normal(gen, dtype, *shape, scale=1.0):
    return (scale * torch.randn(*shape, generator=gen, device="cuda")).to(_TYPES[dtype])


def _cache8(case, gen, n_pages):
    """A full 8-bit cache: pages x kv_heads x slots x head_dim, and its scales, blocks of different loudness."""
    hkv, page, d, block = case["kv_heads"], case["page"], case["head_dim"], case["block"]
    loud = torch.exp2(torch.randn(n_pages, hkv, page // block, 1, 1, generator=gen, device="cuda") * 0.5)
    x = torch.randn(n_pages, hkv, page // block, block, d, generator=gen, device="cuda") * loud
    e = _exponent(x.abs().amax((-1, -2)))
    return (_to_e4m3(x, e[..., None, None]).view(n_pages, hkv, page, d), (e + 127).to(torch.uint8))


def _prepare_batch(case, gen, st):
    hkv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    q, kv = _lengths(case)
    per, n_prefix = -(-max(kv) // page), -(-case["prefix"] // page)
    n_pages = n_prefix + case["batch"] * per
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)  # pages in no order
    start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    st.update(q=q, kv=kv, tokens=int(start[-1]), per=per, q_start=torch.from_numpy(start).cuda(),
              len=torch.tensor(kv, dtype=torch.int32).cuda(), prefix_pages=order[:n_prefix].contiguous(),
              pages=order[n_prefix:].view(case["batch"], per).contiguous())
    st["k_cache"], st["k_scale"] = _cache8(case, gen, n_pages)
    st["v_cache"], st["v_scale"] = _cache8(case, gen, n_pages)
    if case["kind"] == "append":
        # what one projection gives: queries, keys and values of a token side by side
        qkv = _normal(gen, case["dtype"], st["tokens"], case["heads"] + 2 * hkv, d)
        st["q_in"], st["k_in"], st["v_in"] = qkv.split([case["heads"], hkv, hkv], 1)
    else:
        st["q_in"] = _normal(gen, case["dtype"], st["tokens"], case["heads"], d, scale=1.5)
    if own:
        ctx = _ctx()
        import vtq

        st["own_cache"] = vtq.Kv8Cache(st["k_cache"].data_ptr(), st["v_cache"].data_ptr(), st["k_scale"].data_ptr(),
                                       st["v_scale"].data_ptr(), n_pages, page, hkv, d, block=case["block"])
        st["own_batch"] = vtq.KvBatch(case["batch"], st["q_start"].data_ptr(), st["len"].data_ptr(),
                                      st["pages"].data_ptr(), per, max_q=case["q_max"], prefix_len=case["prefix"],
                                      prefix_pages=st["prefix_pages"].data_ptr() if case["prefix"] else None)
        st["y"] = torch.empty(st["tokens"], case["heads"], d, dtype=_TYPES[case["dtype"]], device="cuda")
        if case["kind"] == "append":
            st["rope"] = vtq.Rope(case["rot_dim"], {"half": vtq.ROPE_HALF,
                                                    "interleaved": vtq.ROPE_INTERLEAVED}[case["layout"]])
        else:
            st["lse"] = torch.empty(st["tokens"], case["heads"], dtype=torch.float32, device="cuda")
            need = ctx.kv8_attention_workspace(st["own_cache"], st["own_batch"], _tag(case["dtype"]), st["tokens"],
                                               case["heads"])
            st["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")


def _prepare_beam(case, gen, st):
    rows, vocab, groups = case["groups"] * case["beams"], case["vocab"], case["groups"]
    # peaked rows, as a trained model gives them
    x = torch.randn(rows, vocab, generator=gen, device="cuda") * 2.5
    x[:, torch.randperm(vocab, generator=gen, device="cuda")[: max(1, vocab // 2000)]] += 8.0
    st["logits"] = x.to(_TYPES[case["dtype"]])
    st["score"] = -20.0 * torch.rand(rows, generator=gen, device="cuda")
    st["end"] = 2
    st["done"] = torch.zeros(rows, dtype=torch.uint8, device="cuda")
    st["done"][torch.randperm(rows, generator=gen, device="cuda")[: case["done"]]] = 1
    if own:
        keep = case["keep"]
        st["out"] = (torch.empty(groups, keep, dtype=torch.float32, device="cuda"),
                     torch.empty(groups, keep, dtype=torch.int32, device="cuda"),
                     torch.empty(groups, keep, dtype=torch.int32, device="cuda"),
                     torch.empty(groups, keep, dtype=torch.uint8, device="cuda"))
        need = _ctx().beam_select_workspace(groups, case["beams"], vocab, keep)
        st["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")


def _prepare_pages(case, gen, st):
    batch, most, page, n_pages = case["batch"], case["max_pages"], case["page"], case["n_pages"]
    grow = case["grow"]
    if case["kind"] == "compact":
        # pages in use anywhere in the cache
        share = min(0.98, case["live"] * n_pages / (batch * most))
    else:
        share = min(0.98, (n_pages - 8) / (batch * most + 2.0 * batch * (1 + grow // page)) * 0.9)
    # lengths about a mean that leaves room
    lens = torch.rand(batch, generator=gen, device="cuda") * 0.6 + 0.7
    lens = (lens * share * most * page / 1.3).long().clamp(1, most * page - grow)
    held = (lens + page - 1) // page
    ends = torch.cumsum(held, 0)
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    j = torch.arange(most, device="cuda")[None, :]
    at = (ends - held)[:, None] + j
    st["pages"] = torch.where(j < held[:, None], order[at.clamp(max=n_pages - 1)], -1).to(torch.int32)
    if case["kind"] == "reorder":
        # every second sequence has the first half of its neighbour's pages, from an earlier fork
        whole = (lens // page)
        both = torch.minimum(whole[0::2][: batch // 2], whole[1::2]) // 2
        st["pages"][1::2] = torch.where(j < both[:, None], st["pages"][0::2][: batch // 2], st["pages"][1::2])
    st["len"] = lens.to(torch.int32)
    flat = st["pages"].flatten().long()
    st["refs"] = torch.bincount(flat[flat >= 0], minlength=n_pages).to(torch.int32)
    shape = (case["layers"], n_pages, case["kv_heads"], page, case["head_dim"])
    for name in ("k_cache", "v_cache"):
        if case["cache"] == "e4m3":
            x = torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8).bitwise_and_(0xF7)
            st[name] = x.view(torch.float8_e4m3fn)
        else:
            st[name] = _normal(gen, case["cache"], *shape)
    if case["cache"] == "e4m3":
        for name in ("k_scale", "v_scale"):
            st[name] = torch.randint(118, 126, shape[:3] + (page // 16,), generator=gen, device="cuda",
                                     dtype=torch.uint8)
    if case["kind"] == "reorder":
        i = torch.arange(batch, device="cuda")
        u = torch.rand(batch, generator=gen, device="cuda")
        if case["parents"] == "beams":  # beams of four: the better ones go on more than once
            parent = i // 4 * 4 + (u * u * 4).long()
        else:  # one in ten ends, one in ten forks off another, the rest goes on
            parent = torch.where(u < 0.1, -1, torch.where(u < 0.2, (u * 10 * batch).long() % batch, i))
        st["parent"] = parent.clamp(max=batch - 1).to(torch.int32)
        st["grow"] = torch.full((batch,), grow, dtype=torch.int32, device="cuda")
    # what the calls write
    st["new_pages"], st["new_len"] = torch.empty_like(st["pages"]), torch.empty_like(st["len"])
    st["new_refs"] = torch.empty_like(st["refs"])
    copies = batch if case["kind"] == "reorder" else n_pages // 2
    st["copies"] = torch.empty(copies, 3, dtype=torch.int32, device="cuda")
    st["info"] = torch.empty(2, dtype=torch.int32, device="cuda")
    if own:
        ctx = _ctx()
        import vtq

        if case["cache"] == "e4m3":
            st["own_cache"] = vtq.Kv8Cache(st["k_cache"].data_ptr(), st["v_cache"].data_ptr(),
                                           st["k_scale"].data_ptr(), st["v_scale"].data_ptr(), n_pages, page,
                                           case["kv_heads"], case["head_dim"], block=16)
        else:
            st["own_cache"] = vtq.KvCache(_tag(case["cache"]), st["k_cache"].data_ptr(), st["v_cache"].data_ptr(),
                                          n_pages, page, case["kv_heads"], case["head_dim"])
        need = (ctx.pages_reorder_workspace(n_pages, batch, batch) if case["kind"] == "reorder"
                else ctx.pages_compact_workspace(n_pages))
        st["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = {"case": case}
    {"append": _prepare_batch, "attention": _prepare_batch, "beam": _prepare_beam, "reorder": _prepare_pages,
     "compact": _prepare_pages}[case["kind"]](case, gen, st)
    return st


# ------------------------------------------------------------------ plain forms

def _token_rows(st):
    """Sequence and place among the sequence's own tokens, for every new token."""
    q, kv = torch.tensor(st["q"], device="cuda"), torch.tensor(st["kv"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(st["q"]), device="cuda"), q)
    i = torch.arange(st["tokens"], device="cuda") - (torch.cumsum(q, 0) - q)[seq]
    return seq, (kv - q)[seq] + i


def _scales(st, which):
    return st[which].view(torch.float8_e8m0fnu)


def _into_cache(st, which, x, seq, place):
    """x [tokens, kv_heads, head_dim] in 32 bits into the slots of an 8-bit cache, the earlier tokens of a block to
    its new scale."""
    case = st["case"]
    page, block, hkv, d = case["page"], case["block"], case["kv_heads"], case["head_dim"]
    cache, scale = st[which + "_cache"], st[which + "_scale"]
    per = page // block
    # a block of the cache for every token; tokens of one block share a number
    at = st["pages"][seq, place // page].long() * per + place % page // block
    blocks, mine = torch.unique(at, return_inverse=True)
    top = torch.zeros(len(blocks), hkv, device="cuda")
    size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    top.scatter_reduce_(0, mine[:, None].expand(-1, hkv), size, "amax")
    first = torch.full((len(blocks),), block, device="cuda").scatter_reduce_(0, mine, place % block, "amin")
    p, b = blocks // per, blocks % per
    before = scale[p, :, b].long().clamp(127 + _LEAST, 127 + _MOST) - 127
    e = _exponent(top)
    e = torch.where(first[:, None] > 0, torch.maximum(e, before), e)
    slots = b[:, None] * block + torch.arange(block, device="cuda")[None, :]
    bits = cache.view(torch.uint8)
    old = bits[p[:, None], :, slots].view(torch.float8_e4m3fn).float()  # [blocks, slots, heads, d]
    turned = _to_e4m3(torch.ldexp(old, before[:, None, :, None]), e[:, None, :, None])
    earlier = torch.arange(block, device="cuda")[None, :] < first[:, None]
    bits[p[:, None], :, slots] = torch.where(earlier[:, :, None, None], turned.view(torch.uint8),
                                             bits[p[:, None], :, slots])
    bits[p[mine], :, place % page] = _to_e4m3(x, e[mine][..., None]).view(torch.uint8)
    scale[p, :, b] = (e + 127).to(torch.uint8)


def _plain_append(st):
    case = st["case"]
    seq, place = _token_rows(st)
    _into_cache(st, "k", _rotate(case, st["k_in"], place + case["prefix"]), seq, place)
    _into_cache(st, "v", st["v_in"].float(), seq, place)
    y = _rotate(case, st["q_in"], place + case["prefix"]).to(_TYPES[case["dtype"]])
    return y, st["k_cache"], st["v_cache"], _scales(st, "k_scale"), _scales(st, "v_scale")


def _widened(st, which, pages):
    """Pages of the cache as the values they stand for, in 32 bits."""
    case = st["case"]
    x = st[which + "_cache"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()
    e = st[which + "_scale"][pages].to(torch.int32) - 127
    return torch.ldexp(x, e.repeat_interleave(case["block"], -1)[..., None])


def _plain_attention(st):
    case = st["case"]
    hkv, d, page, batch = case["kv_heads"], case["head_dim"], case["page"], case["batch"]
    group, prefix, most = case["heads"] // hkv, case["prefix"], max(st["kv"])
    tokens = st["tokens"]
    q = st["q_in"].float().view(tokens, hkv, group, d) * (1.0 / math.sqrt(d))
    seq, place = _token_rows(st)
    # every row against the prefix: [hkv, tokens * group, prefix]
    rows = q.permute(1, 0, 2, 3).reshape(hkv, tokens * group, d)
    pk = _widened(st, "k", st["prefix_pages"].long()).permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :prefix]
    pv = _widened(st, "v", st["prefix_pages"].long()).permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :prefix]
    sp = torch.matmul(rows, pk.transpose(1, 2).contiguous())
    # every sequence's rows, padded, against its own keys, padded: [batch, hkv, q_max * group, most]
    own_pages = st["pages"].long()[:, : -(-most // page)]
    ok = _widened(st, "k", own_pages).permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)[:, :, :most]
    ov = _widened(st, "v", own_pages).permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)[:, :, :most].contiguous()
    first = torch.tensor([0] + list(np.cumsum(st["q"])[:-1]), device="cuda")
    i = torch.arange(tokens, device="cuda") - first[seq]
    padded = torch.zeros(batch, case["q_max"], hkv, group, d, device="cuda")
    padded[seq, i] = q
    so = torch.matmul(padded.permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d), ok.transpose(2, 3).contiguous())
    seen = torch.full((batch, case["q_max"]), -1, dtype=torch.long, device="cuda")
    seen[seq, i] = place
    hidden = torch.arange(most, device="cuda")[None, None, :] > seen[:, :, None]
    so = so.view(batch, hkv, case["q_max"], group, most).masked_fill(hidden[:, None, :, None, :], -math.inf)
    top = so.amax(-1)[seq, :, i]  # [tokens, hkv, group]
    if prefix:
        top = torch.maximum(top, sp.amax(-1).view(hkv, tokens, group).permute(1, 0, 2))
    shift = torch.zeros(batch, case["q_max"], hkv, group, device="cuda")
    shift[seq, i] = top
    po = torch.exp(so - shift.permute(0, 2, 1, 3)[..., None])
    total = po.sum(-1)[seq, :, i]
    out = torch.matmul(po.view(batch, hkv, -1, most), ov).view(batch, hkv, case["q_max"], group, d)[seq, :, i]
    if prefix:
        pp = torch.exp(sp - top.permute(1, 0, 2).reshape(hkv, -1, 1))
        total = total + pp.sum(-1).view(hkv, tokens, group).permute(1, 0, 2)
        out = out + torch.matmul(pp, pv.contiguous()).view(hkv, tokens, group, d).permute(1, 0, 2, 3)
    y = (out / total[..., None]).reshape(tokens, case["heads"], d)
    return y.to(_TYPES[case["dtype"]]), (top + torch.log(total)).reshape(tokens, case["heads"])


def _plain_beam(st):
    case = st["case"]
    groups, beams, vocab, keep = case["groups"], case["beams"], case["vocab"], case["keep"]
    # 64 bits: which of two nearly equal sums is the greater decides about tokens
    x = st["logits"].double()
    top = x.amax(1, keepdim=True)
    norm = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    s = st["score"].double()[:, None] + (x - norm)
    s = torch.where(torch.isnan(s) | torch.isinf(s), -1e300, s)  # counts as -infinity, but is a candidate
    done = st["done"] != 0
    ended = torch.full((1, vocab), -math.inf, dtype=torch.float64, device="cuda").expand(groups * beams, -1).clone()
    ended[:, st["end"]] = st["score"].double()
    s = torch.where(done[:, None], ended, s).view(groups, beams * vocab)
    # the keep greatest of a group, of equal ones those of the lowest indexes
    last = torch.topk(s, keep, 1).values[:, -1:]
    more, equal = s > last, s == last
    taken = more | (equal & (torch.cumsum(equal, 1) <= keep - more.sum(1, keepdim=True)))
    index = taken.nonzero()[:, 1].view(groups, keep)
    order = torch.sort(torch.gather(s, 1, index), dim=1, descending=True, stable=True)
    index = torch.gather(index, 1, order.indices)
    token = index % vocab
    parent = index // vocab + torch.arange(groups, device="cuda")[:, None] * beams
    ends = done[parent] | (token == st["end"])
    none = order.values == -math.inf
    return (order.values.float(), torch.where(none, -1, token).to(torch.int32),
            torch.where(none, -1, parent).to(torch.int32), (ends | none).to(torch.uint8))


def _copy_pages(st, source, target, slots):
    """The first slots of pages, on every layer."""
    page = st["case"]["page"]
    there = torch.arange(page, device="cuda")[None, :] < slots[:, None]
    for name in ("k_cache", "v_cache"):
        x = st[name].view(torch.uint8) if st["case"]["cache"] == "e4m3" else st[name]
        x[:, target] = torch.where(there[None, :, None, :, None], x[:, source], x[:, target])
    if st["case"]["cache"] == "e4m3":
        for name in ("k_scale", "v_scale"):
            x = st[name]
            x[:, target] = torch.where(there[:, ::16][None, :, None, :], x[:, source], x[:, target])


def _page_outputs(st, *more):
    out = [*more, st["k_cache"], st["v_cache"]]
    if st["case"]["cache"] == "e4m3":
        out += [_scales(st, "k_scale"), _scales(st, "v_scale")]
    return out


def _plain_reorder(st):
    case = st["case"]
    page, most, n_pages, batch = case["page"], case["max_pages"], case["n_pages"], case["batch"]
    refs, parent = st["refs"].long(), st["parent"].long()
    has = parent >= 0
    from_ = parent.clamp(min=0)
    lens = torch.where(has, st["len"].long()[from_], 0)
    rows = torch.where(has[:, None], st["pages"].long()[from_], -1)
    whole, used = lens // page, (lens + page - 1) // page
    needed = ((lens + st["grow"].long() + page - 1) // page).clamp(max=most)
    # the first of a parent's children keeps what the parent alone holds
    i = torch.arange(batch, device="cuda")
    first = torch.full((batch,), batch, device="cuda").scatter_reduce_(0, from_, torch.where(has, i, batch), "amin")
    eldest = has & (first[from_] == i)
    j = torch.arange(most, device="cuda")[None, :]
    alone = (rows >= 0) & (refs[rows.clamp(min=0)] == 1) & eldest[:, None] & (j < needed[:, None])
    kept = torch.cumprod((alone | (j < whole[:, None])).long(), 1).bool() & (j >= whole[:, None])
    begin = whole + kept.sum(1)  # fresh pages from here on
    fresh = (j >= begin[:, None]) & (j < needed[:, None])
    table = torch.where((j < whole[:, None]) | kept, rows, -1)
    # the lowest free pages, in the order of sequences and places
    free = torch.sort((refs != 0).long(), stable=True).indices
    count = (refs == 0).sum()
    rank = torch.cumsum(fresh.flatten(), 0).view(batch, most) - 1
    got = fresh & (rank < count)
    table = torch.where(got, free[rank.clamp(0, n_pages - 1)], table)
    uses = torch.zeros(n_pages + 1, dtype=torch.long, device="cuda")
    uses.scatter_add_(0, torch.where(table >= 0, table, n_pages).flatten(), torch.ones_like(table).flatten())
    old = st["pages"].long()
    uses.scatter_add_(0, torch.where(old >= 0, old, n_pages).flatten(), -torch.ones_like(old).flatten())
    st["new_refs"].copy_(refs + uses[:n_pages])
    st["new_pages"].copy_(table)
    st["new_len"].copy_(lens)
    # a part-filled page that others hold too is copied
    at = whole.clamp(max=most - 1)[:, None]
    copied = (begin == whole) & (lens % page > 0) & got.gather(1, at)[:, 0] & (rows.gather(1, at)[:, 0] >= 0)
    which = copied.nonzero()[:, 0]
    source, target, slots = rows.gather(1, at)[which, 0], table.gather(1, at)[which, 0], (lens % page)[which]
    st["copies"].fill_(-1)
    st["copies"][: len(which)] = torch.stack([source, target, slots], 1).to(torch.int32)
    st["info"][0] = len(which)
    st["info"][1] = (fresh.sum() - got.sum()) + (((lens + st["grow"].long() + page - 1) // page) - needed).sum()
    _copy_pages(st, source, target, slots)
    return _page_outputs(st, st["new_pages"], st["new_len"], st["new_refs"], st["copies"], st["info"])


def _plain_compact(st):
    n_pages, page = st["case"]["n_pages"], st["case"]["page"]
    live = st["refs"] > 0
    n_live = live.sum()
    i = torch.arange(n_pages, device="cuda")
    target, source = (~live & (i < n_live)).nonzero()[:, 0], (live & (i >= n_live)).nonzero()[:, 0]
    goes = i.clone()
    goes[source] = target
    st["new_pages"].copy_(torch.where(st["pages"] >= 0, goes[st["pages"].long().clamp(min=0)], -1))
    st["new_refs"].copy_(torch.where(live & (i < n_live), st["refs"], 0))
    st["new_refs"][target] = st["refs"][source]
    slots = torch.full_like(source, page)
    st["copies"].fill_(-1)
    st["copies"][: len(source)] = torch.stack([source, target, slots], 1).to(torch.int32)
    st["info"][0], st["info"][1] = len(source), n_live
    _copy_pages(st, source, target, slots)
    return _page_outputs(st, st["new_pages"], st["new_refs"], st["copies"], st["info"])


# ------------------------------------------------------------------ the library's operators

def _library(st):
    case, ctx = st["case"], _ctx()
    stream = torch.cuda.current_stream().cuda_stream
    kind = case["kind"]
    if kind == "append":
        q, k, v, y = st["q_in"], st["k_in"], st["v_in"], st["y"]
        ctx.kv8_append_device(st["own_cache"], st["own_batch"], st["rope"], _tag(case["dtype"]), st["tokens"],
                              k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), stream,
                              heads=case["heads"], q_ptr=q.data_ptr(), q_token_stride=q.stride(0),
                              q_head_stride=q.stride(1), q_out_ptr=y.data_ptr(), q_out_token_stride=y.stride(0),
                              q_out_head_stride=y.stride(1))
        return y, st["k_cache"], st["v_cache"], _scales(st, "k_scale"), _scales(st, "v_scale")
    if kind == "attention":
        q, y = st["q_in"], st["y"]
        ctx.kv8_attention_device(st["own_cache"], st["own_batch"], _tag(case["dtype"]), st["tokens"], case["heads"],
                                 q.data_ptr(), q.stride(0), q.stride(1), y.data_ptr(), y.stride(0), y.stride(1),
                                 1.0 / math.sqrt(case["head_dim"]), st["ws"].data_ptr(), st["ws"].numel(), stream,
                                 lse_ptr=st["lse"].data_ptr())
        return y, st["lse"]
    if kind == "beam":
        score, token, parent, done = st["out"]
        ctx.beam_select_device(_tag(case["dtype"]), st["logits"].data_ptr(), case["vocab"], case["groups"],
                               case["beams"], case["vocab"], st["score"].data_ptr(), case["keep"], score.data_ptr(),
                               token.data_ptr(), parent.data_ptr(), st["ws"].data_ptr(), st["ws"].numel(), stream,
                               done_ptr=st["done"].data_ptr(), end_token=st["end"], out_done_ptr=done.data_ptr())
        return score, token, parent, done
    n_pages, page, batch = case["n_pages"], case["page"], case["batch"]
    if kind == "reorder":
        ctx.pages_reorder_device(n_pages, page, case["max_pages"], st["refs"].data_ptr(), batch,
                                 st["pages"].data_ptr(), st["len"].data_ptr(), batch, st["parent"].data_ptr(),
                                 st["grow"].data_ptr(), st["new_refs"].data_ptr(), st["new_pages"].data_ptr(),
                                 st["new_len"].data_ptr(), st["copies"].data_ptr(), st["info"].data_ptr(),
                                 st["ws"].data_ptr(), st["ws"].numel(), stream)
    else:
        ctx.pages_compact_device(n_pages, page, st["refs"].data_ptr(), batch * case["max_pages"],
                                 st["pages"].data_ptr(), st["new_refs"].data_ptr(), st["new_pages"].data_ptr(),
                                 st["copies"].data_ptr(), st["info"].data_ptr(), st["ws"].data_ptr(),
                                 st["ws"].numel(), stream)
    x = st["k_cache"]
    ctx.pages_copy_device(st["own_cache"], case["layers"], x.stride(0), st["copies"].data_ptr(),
                          st["copies"].shape[0], st["info"].data_ptr(), stream,
                          scale_layer_stride=st["k_scale"].stride(0) if case["cache"] == "e4m3" else 0)
    if kind == "reorder":
        return _page_outputs(st, st["new_pages"], st["new_len"], st["new_refs"], st["copies"], st["info"])
    return _page_outputs(st, st["new_pages"], st["new_refs"], st["copies"], st["info"])


def run(state):
    if own:
        return _library(state)
    return {"append": _plain_append, "attention": _plain_attention, "beam": _plain_beam, "reorder": _plain_reorder,
            "compact": _plain_compact}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ work and exact results

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
    if case["kind"] == "beam":
        rows = case["groups"] * case["beams"]
        return {"bytes": (rows - case["done"]) * case["vocab"] * size[case["dtype"]] + 5 * rows
                + 13 * case["groups"] * case["keep"], "flops": 4 * (rows - case["done"]) * case["vocab"]}
    if case["kind"] in ("reorder", "compact"):
        # tables and counts in and out, and what is copied, on the mean over inputs
        batch, page = case["batch"], case["page"]
        bytes_ = 8 * batch * case["max_pages"] + 8 * case["n_pages"] + 8 * batch
        slot = 2 * case["layers"] * case["kv_heads"] * (case["head_dim"] * size[case["cache"]])
        if case["kind"] == "compact":
            live = min(case["live"], 0.98 * batch * case["max_pages"] / case["n_pages"]) / 1.3
            moved = live * (1 - live) * case["n_pages"]
            return {"bytes": bytes_ + 12 * moved + 2 * moved * page * slot, "flops": 0}
        # of four beams with u^2 4 the parents, 1.7 are second children; one in ten forks besides
        copied = batch * (0.43 if case["parents"] == "beams" else 0.1)
        return {"bytes": bytes_ + 12 * copied + copied * page * slot, "flops": 0}
    q, kv = _lengths(case)
    tokens, d = sum(q), case["head_dim"]
    if case["kind"] == "append":
        cached = tokens * 2 * case["kv_heads"] * d
        return {"bytes": 2 * tokens * case["heads"] * d * size[case["dtype"]] + cached * (size[case["dtype"]] + 1)
                + cached // (d * min(case["block"], case["q_max"])) + 4 * (3 * case["batch"] + 1),
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rot_dim"]}
    keys = sum(n * case["prefix"] + n * (m - n) + n * (n + 1) // 2 for n, m in zip(q, kv))
    cached = (case["prefix"] + sum(kv)) * 2 * case["kv_heads"]
    return {"bytes": cached * d + cached // case["block"] + 2 * tokens * case["heads"] * d * size[case["dtype"]]
            + 4 * tokens * case["heads"], "flops": 4 * case["heads"] * d * keys}


def _exact_rotate(case, x, pos):
    """Complex rotation of x [tokens, heads, head_dim] by pos in 64 bits."""
    r = case["rot_dim"]
    f = torch.tensor([10000.0 ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64, device=x.device)
    angle = (pos.double().unsqueeze(1) * f.unsqueeze(0)).unsqueeze(1)
    turn = torch.polar(torch.ones_like(angle), angle)
    x = x.double()
    head = x[..., :r]
    if case["layout"] == "half":
        z = torch.complex(head[..., : r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
        rotated = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], r // 2, 2).contiguous()) * turn
        rotated = torch.view_as_real(z).reshape(head.shape)
    return torch.cat([rotated, x[..., r:]], -1)


def _exact_append(case, st):
    page, block, prefix = case["page"], case["block"], case["prefix"]
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(st["q"], st["kv"])]).cuda() + prefix
    new = {"k": _exact_rotate(case, st["k_in"], pos), "v": st["v_in"].double()}
    out = [_exact_rotate(case, st["q_in"], pos)]
    codes, scales = [], []
    for which in ("k", "v"):
        cache, scale = st[which + "_cache"].double(), st[which + "_scale"].double() - 127.0
        t = 0
        for b, (n, m) in enumerate(zip(st["q"], st["kv"])):
            place = m - n
            while place < m:
                stop = min(m, place // block * block + block)
                p, s0, s1 = int(st["pages"][b, place // page]), place % page, place % page + stop - place
                group = s0 // block
                x = new[which][t:t + stop - place].transpose(0, 1)  # heads x tokens x elements
                e = torch.ceil(torch.log2(x.abs().flatten(1).amax(1) / 448.0))
                if s0 % block:
                    e = torch.maximum(e, scale[p, :, group])
                    cache[p, :, group * block:s0] *= torch.exp2(scale[p, :, group] - e)[:, None, None]
                cache[p, :, s0:s1] = x * torch.exp2(-e)[:, None, None]
                scale[p, :, group] = e
                t, place = t + stop - place, stop
        codes.append(cache)
        scales.append(torch.exp2(scale))
    return out + codes + scales


def _exact_attention(case, st):
    page, prefix, block = case["page"], case["prefix"], case["block"]
    begin = [0]
    for n in st["q"]:
        begin.append(begin[-1] + n)
    d, group = case["head_dim"], case["heads"] // case["kv_heads"]
    value = {}
    for which in ("k", "v"):
        x = st[which + "_cache"].double().unflatten(2, (page // block, block))
        value[which] = (x * torch.exp2(st[which + "_scale"].double() - 127.0)[..., None, None]).flatten(2, 3)
    ys, ls = [], []
    for b, (n, m) in enumerate(zip(st["q"], st["kv"])):
        def sequence(which):
            """[kv_heads, prefix + m, head_dim]"""
            own_part = value[which][st["pages"][b].long()].transpose(0, 1).flatten(1, 2)[:, :m]
            shared = value[which][st["prefix_pages"].long()].transpose(0, 1).flatten(1, 2)[:, :prefix]
            return torch.cat([shared, own_part], 1)
        q = st["q_in"][begin[b]:begin[b + 1]].double().unflatten(1, (-1, group)).permute(1, 2, 0, 3).flatten(1, 2)
        score = torch.bmm(q, sequence("k").transpose(1, 2).contiguous()) / math.sqrt(d)
        last = prefix + m - n + torch.arange(n, device="cuda")
        after = torch.arange(prefix + m, device="cuda")[None, :] > last[:, None]
        score = score.unflatten(1, (group, n)).masked_fill(after, -math.inf)
        norm = torch.logsumexp(score, -1)
        weight = torch.exp(score - norm[..., None]).flatten(1, 2)
        y = torch.bmm(weight, sequence("v")).unflatten(1, (group, n))
        ys.append(y.permute(2, 0, 1, 3).reshape(n, case["heads"], d))
        ls.append(norm.permute(2, 0, 1).reshape(n, case["heads"]))
    return torch.cat(ys), torch.cat(ls)


def _exact_beam(case, st):
    beams, vocab, keep = case["beams"], case["vocab"], case["keep"]
    got = []
    for g in range(case["groups"]):
        rows = slice(g * beams, (g + 1) * beams)
        s = torch.log_softmax(st["logits"][rows].double(), -1) + st["score"][rows].double().unsqueeze(1)
        ended = st["done"][rows].bool()
        live = s[~ended].flatten()
        missing = torch.full((keep,), -math.inf, dtype=torch.float64, device="cuda")
        every = torch.cat([live, st["score"][rows][ended].double(), missing])
        got.append(every.sort(descending=True).values[:keep])
    return torch.stack(got), None, None, None


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, st)
    if case["kind"] == "beam":
        return _exact_beam(case, st)
    if case["kind"] == "attention":
        return None if work(case)["flops"] > 2e12 else _exact_attention(case, st)
    # page by page: what the lists of a run say, the caches as they then are
    lists = _serial_reorder(case, st) if case["kind"] == "reorder" else _serial_compact(case, st)
    values = {n: st[n].double() for n in ("k_cache", "v_cache")}
    scales = {n: torch.exp2(st[n].double() - 127.0) for n in ("k_scale", "v_scale") if n in st}
    for source, target, slots in lists.pop():
        for x in values.values():
            x[:, target, :, :slots] = x[:, source, :, :slots].clone()
        for x in scales.values():
            x[:, target, :, : -(-slots // 16)] = x[:, source, :, : -(-slots // 16)].clone()
    return lists + list(values.values()) + list(scales.values())


def _serial_reorder(case, st):
    """The lists of a reorder, one sequence after another: five that hold no computed numbers, and the copies."""
    page, most = case["page"], case["max_pages"]
    refs, table, lens = st["refs"].tolist(), st["pages"].tolist(), st["len"].tolist()
    free = [p for p, r in enumerate(refs) if r == 0]
    seen, copies = set(), []
    for parent in st["parent"].tolist():
        row, n = (table[parent], lens[parent]) if parent >= 0 else ([-1] * most, 0)
        at = n // page
        needed = min(most, -(-(n + case["grow"]) // page))
        if parent >= 0 and parent not in seen:
            while at < needed and row[at] >= 0 and refs[row[at]] == 1:
                at += 1
        seen.add(parent)
        for j in range(at, needed):
            if free:
                p = free.pop(0)
                if j == n // page and n % page and row[j] >= 0:
                    copies.append((row[j], p, n % page))
    return [None] * 5 + [copies]


def _serial_compact(case, st):
    refs = st["refs"].tolist()
    live = [p for p, r in enumerate(refs) if r]
    high = [p for p in live if p >= len(live)]
    low = [p for p in range(len(live)) if refs[p] == 0]
    return [None] * 4 + [[(s, t, case["page"]) for s, t in zip(high, low)]]
