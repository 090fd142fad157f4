"""Performance cases of the batched serving operators: int8 linear, rotary positions, paged KV append, attention
over a shared prefix.

A case is one of
  i8         activations quantized to 8 bits a token, then the product with 8-bit weights scaled a channel;
  rope       rotary positions on the heads of a batch of tokens;
  append     a step's keys (rotated), values (as they are) and queries (rotated) of a ragged batch, keys and
             values into a paged cache;
  attention  a ragged batch against a prefix that all sequences share and the pages of their own.

`run` computes a case in elementary torch operations, or, where `own` is set, through the library.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _i8(m, k, n, dtype, out, bias=False):
    return {"kind": "i8", "tokens": m, "in_feat": k, "out_feat": n, "dtype": dtype, "out": out, "bias": bias}


def _rope(tokens, heads, head_dim, rot_dim, layout, scaling, first, dtype, theta=10000.0, factor=1.0, original=4096):
    return {"kind": "rope", "tokens": tokens, "heads": heads, "head_dim": head_dim, "rot_dim": rot_dim,
            "layout": layout, "scaling": scaling, "factor": factor, "original": original, "theta": theta,
            "first": first, "dtype": dtype}


def _append(batch, q_max, prefix, own_max, heads, kv_heads, head_dim, rot_dim, layout, page, dtype, cache, ragged):
    return {"kind": "append", "batch": batch, "q_max": q_max, "prefix": prefix, "own_max": own_max, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "rot_dim": rot_dim, "layout": layout, "page": page,
            "dtype": dtype, "cache": cache, "ragged": ragged}


def _attention(batch, q_max, prefix, own_max, heads, kv_heads, head_dim, page, dtype, cache, ragged):
    return {"kind": "attention", "batch": batch, "q_max": q_max, "prefix": prefix, "own_max": own_max, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "cache": cache, "ragged": ragged}


def listed():
    return [
        # one token through an attention-sized matrix of a 7B model
        {"name": "i8_decode_4096", **_i8(1, 4096, 4096, "bf16", "bf16")},
        # nineteen sequences decoded together, down projection, f32 as the other linears give it, with a bias
        {"name": "i8_batch19_down", **_i8(19, 11008, 4096, "f32", "f32", True)},
        # a prompt of 512 tokens, up projection of an 8B model
        {"name": "i8_prompt512_up", **_i8(512, 4096, 14336, "bf16", "bf16")},
        # prompts of several sequences packed together, a token count that no tile divides
        {"name": "i8_packed4001_up", **_i8(4001, 4096, 11008, "f16", "f16")},
        # eight sequences of the 1.1B model decoded together, its rotation
        {"name": "rope_decode8", **_rope(8, 36, 64, 64, "interleaved", "none", 700, "f32")},
        # a long prompt's queries and keys far into a scaled context
        {"name": "rope_prompt4096_yarn", **_rope(4096, 40, 128, 128, "half", "yarn", 126000, "bf16", 1e6, 16.0, 8192)},
        # 32 sequences, one new token each, behind a shared system prompt
        {"name": "append_decode32", **_append(32, 1, 2048, 700, 32, 8, 128, 128, "half", 16, "bf16", "bf16", 11)},
        # packed prompts of five sequences, part of each head rotated, f32 activations into a 16-bit cache
        {"name": "append_prompts", **_append(5, 1200, 0, 1200, 32, 8, 80, 32, "interleaved", 64, "f32", "f16", 12)},
        # four sequences of the 1.1B model, all in f32
        {"name": "attention_decode4_f32", **_attention(4, 1, 500, 90, 32, 4, 64, 16, "f32", "f32", 13)},
        # drafts of up to six tokens to be checked at once, odd lengths, a short prefix
        {"name": "attention_drafts16", **_attention(16, 6, 1003, 4000, 24, 8, 96, 32, "f16", "f16", 14)},
        # 64 chats behind a system prompt of 8192 tokens
        {"name": "attention_batch64_8k", **_attention(64, 1, 8192, 512, 32, 8, 128, 16, "bf16", "bf16", 15)},
        # 128 questions about one document
        {"name": "attention_batch128_32k", **_attention(128, 1, 32768, 1024, 32, 8, 128, 64, "bf16", "bf16", 16)},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One more case: any of the four kinds, their types and layouts, sizes over the listed ranges."""
    kind = rng.choice(["i8", "i8", "rope", "append", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "i8":
        while True:
            m = 1 if rng.random() < 0.25 else _log_int(rng, 2, 4096)
            k, n = _log_int(rng, 100, 14336), _log_int(rng, 64, 32000)
            if rng.random() < 0.7:  # most matrices have whole multiples of 64
                k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
            if m * k * n <= 4001 * 4096 * 11008:
                return _i8(m, k, n, dtype, rng.choice([dtype, "f32"]), rng.random() < 0.3)
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    group = rng.choice([1, 2, 4, 4, 7, 8])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * group
    page = rng.choice([16, 16, 32, 64, 128])
    layout = rng.choice(["interleaved", "half"])
    rot = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
    if kind == "rope":
        most = 4096 * 40 * 128
        tokens = min(_log_int(rng, 1, 8192), most // (heads * head_dim))
        scaling = rng.choice(["none", "none", "linear", "bands", "yarn"])
        return _rope(tokens, heads, head_dim, rot, layout, scaling, _log_int(rng, 1, 500000), dtype,
                     rng.choice([10000.0, 500000.0, 1e6]), 1.0 if scaling == "none" else rng.choice([2.0, 8.0, 16.0]),
                     rng.choice([2048, 4096, 8192]))
    cache = dtype if dtype != "f32" else rng.choice(["f32", "f32", "f16", "bf16"])
    ragged = rng.randint(100, 10 ** 6)
    if kind == "append":
        q_max = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1200)
        batch = max(1, min(_log_int(rng, 1, 128), 5000 // q_max))
        return _append(batch, q_max, _log_int(rng, 1, 32768), q_max + _log_int(rng, 1, 2000), heads, kv_heads, head_dim,
                       rot, layout, page, dtype, cache, ragged)
    while True:
        q_max = 1 if rng.random() < 0.5 else _log_int(rng, 2, 300)
        batch = _log_int(rng, 1, 128)
        prefix = 0 if rng.random() < 0.15 else _log_int(rng, 16, 32768)
        own_max = q_max + _log_int(rng, 1, 4000)
        rows = batch * q_max * heads
        most = 128 * 32 * (32768 + 1024) * 128
        if dtype == "f32":  # the f32 matrix rate is a sixteenth of the 16-bit one
            most //= 8
        if rows * (prefix + own_max) * head_dim <= most and batch * own_max * kv_heads * head_dim <= 1 << 27:
            return _attention(batch, q_max, prefix, own_max, heads, kv_heads, head_dim, page, dtype, cache, ragged)


# ------------------------------------------------------------------ lengths, pages

def _lengths(case):
    """New tokens and cached own tokens (the new ones among them) of every sequence."""
    rng = random.Random(case["ragged"])
    q = [rng.randint((case["q_max"] + 1) // 2, case["q_max"]) for _ in range(case["batch"])]
    q[0] = case["q_max"]
    kv = [n + rng.randint((case["own_max"] - case["q_max"]) // 2, case["own_max"] - case["q_max"]) for n in q]
    return q, kv


def _turn_angles(case, pos):
    """Angles [tokens, pairs] in 64 bits and the magnitude of the rotation."""
    r, theta = case["rot_dim"], case.get("theta", 10000.0)
    s, scaling, original = case.get("factor", 1.0), case.get("scaling", "none"), case.get("original", 4096)
    i = torch.arange(r // 2, dtype=torch.float64, device=pos.device)
    f = torch.exp(-2.0 * i / r * math.log(theta))
    magnitude = 1.0
    if scaling == "linear":
        f = f / s
    elif scaling == "bands":
        # turns within the original context: few are stretched, many are kept
        keep = ((original * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = keep * f + (1 - keep) * f / s
    elif scaling == "yarn":
        lo = max(0, math.floor(r * math.log(original / (32.0 * 2 * math.pi)) / (2 * math.log(theta))))
        hi = min(r - 1, math.ceil(r * math.log(original / (1.0 * 2 * math.pi)) / (2 * math.log(theta))))
        stretch = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = (1 - stretch) * f + stretch * f / s
        magnitude = 0.1 * math.log(s) + 1.0
    return pos.double()[:, None] * f[None, :], magnitude


def _rotate(case, x, angles, magnitude):
    """x [tokens, heads, head_dim] in 32 bits."""
    r = case["rot_dim"]
    c = (torch.cos(angles) * magnitude).float()[:, None, :]
    s = (torch.sin(angles) * magnitude).float()[:, None, :]
    x = x.float()
    out = x.clone()
    if case["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        out[..., : r // 2], out[..., r // 2: r] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2], out[..., 1:r:2] = a * c - b * s, a * s + b * c
    return out


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


def _up16(n):
    return (n + 15) // 16 * 16


def _rope_plan(case):
    import vtq

    return vtq.Rope(case["rot_dim"], {"half": vtq.ROPE_HALF, "interleaved": vtq.ROPE_INTERLEAVED}[case["layout"]],
                    theta=case.get("theta", 10000.0),
                    scaling={"none": vtq.ROPE_SCALE_NONE, "linear": vtq.ROPE_SCALE_LINEAR,
                             "bands": vtq.ROPE_SCALE_BANDS, "yarn": vtq.ROPE_SCALE_YARN}[case.get("scaling", "none")],
                    factor=case.get("factor", 1.0), original_context=case.get("original", 4096))


def _paged(case, gen):
    """The ragged batch's device arrays and an empty cache that holds it, its pages in no order."""
    q, kv = _lengths(case)
    page, prefix = case["page"], case["prefix"]
    per = -(-max(kv) // page)
    n_prefix = -(-prefix // page)
    n_pages = n_prefix + case["batch"] * per
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    st = {"q": q, "kv": kv, "tokens": int(start[-1]), "n_pages": n_pages, "per": per,
          "q_start": torch.from_numpy(start).cuda(), "len": torch.tensor(kv, dtype=torch.int32).cuda(),
          "prefix_pages": order[:n_prefix].contiguous(),
          "pages": order[n_prefix:].view(case["batch"], per).contiguous()}
    return st


def _library_batch(case, st):
    import vtq

    st["own_cache"] = vtq.KvCache(_tag(case["cache"]), st["k_cache"].data_ptr(), st["v_cache"].data_ptr(),
                                  st["n_pages"], case["page"], case["kv_heads"], case["head_dim"])
    st["own_batch"] = vtq.KvBatch(case["batch"], st["q_start"].data_ptr(), st["len"].data_ptr(),
                                  st["pages"].data_ptr(), st["per"], max_q=case["q_max"], prefix_len=case["prefix"],
                                  prefix_pages=st["prefix_pages"].data_ptr() if case["prefix"] else None)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = {"case": case}
    if case["kind"] == "i8":
        m, k, n = case["tokens"], case["in_feat"], case["out_feat"]
        x = torch.randn(m, k, generator=gen, device="cuda")
        x[:, torch.randperm(k, generator=gen, device="cuda")[: max(1, k // 256)]] *= 8.0  # a few loud channels
        st["x"] = x.to(_TYPES[case["dtype"]])
        w = torch.randn(n, k, generator=gen, device="cuda") * 0.02
        ws = w.abs().amax(1) / 127
        st["w"] = torch.zeros(n, _up16(k), dtype=torch.int8, device="cuda")  # rows start at multiples of 16 bytes
        st["w"][:, :k] = torch.round(w / ws[:, None]).to(torch.int8)
        st["ws"] = ws
        st["bias"] = torch.randn(n, generator=gen, device="cuda") * 0.1 if case["bias"] else None
        if own:
            _ctx()
            st["xq"] = torch.empty(m, _up16(k), dtype=torch.int8, device="cuda")
            st["xs"] = torch.empty(m, dtype=torch.float32, device="cuda")
            st["y"] = torch.empty(m, n, dtype=_TYPES[case["out"]], device="cuda")
    elif case["kind"] == "rope":
        st["x"] = _normal(gen, case["dtype"], case["tokens"], case["heads"], case["head_dim"])
        shift = int(torch.randint(0, 64, (1,), generator=gen, device="cuda"))
        st["pos"] = torch.arange(case["tokens"], dtype=torch.int32, device="cuda") + (case["first"] + shift)
        if own:
            _ctx()
            st["rope"] = _rope_plan(case)
            st["y"] = torch.empty_like(st["x"])
    else:
        hkv, d = case["kv_heads"], case["head_dim"]
        st.update(_paged(case, gen))
        shape = (st["n_pages"], hkv, case["page"], d)
        if case["kind"] == "append":
            # what one projection gives: queries, keys and values of a token side by side
            qkv = _normal(gen, case["dtype"], st["tokens"], case["heads"] + 2 * hkv, d)
            st["q_in"], st["k_in"], st["v_in"] = qkv.split([case["heads"], hkv, hkv], 1)
            st["k_cache"] = torch.zeros(shape, dtype=_TYPES[case["cache"]], device="cuda")
            st["v_cache"] = torch.zeros(shape, dtype=_TYPES[case["cache"]], device="cuda")
        else:
            st["q_in"] = _normal(gen, case["dtype"], st["tokens"], case["heads"], d, scale=1.5)
            st["k_cache"] = _normal(gen, case["cache"], *shape)
            st["v_cache"] = _normal(gen, case["cache"], *shape)
        if own:
            ctx = _ctx()
            _library_batch(case, st)
            st["y"] = torch.empty(st["tokens"], case["heads"], d, dtype=_TYPES[case["dtype"]], device="cuda")
            if case["kind"] == "append":
                st["rope"] = _rope_plan(case)
            else:
                st["lse"] = torch.empty(st["tokens"], case["heads"], dtype=torch.float32, device="cuda")
                need = ctx.attention_workspace(st["own_cache"], st["own_batch"], _tag(case["dtype"]), st["tokens"],
                                               case["heads"])
                st["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return st


# ------------------------------------------------------------------ plain forms

def _plain_i8(st):
    case, x = st["case"], st["x"].float()
    k = case["in_feat"]
    scale = (x.abs().amax(1).double() / 127.0).float()
    # the quotient in 64 bits: in 32 it rounds onto a half now and then
    q = torch.round(x.double() / torch.where(scale > 0, scale, 1.0).double()[:, None]).float()
    acc = None
    for k0 in range(0, k, 1024):  # 1024 products of 127 * 127 stay below 2^24: sums in 32 bits are exact
        k1 = min(k, k0 + 1024)
        part = (q[:, k0:k1] @ st["w"][:, k0:k1].float().t()).to(torch.int32)
        acc = part if acc is None else acc + part
    y = acc.float() * scale[:, None] * st["ws"][None, :]
    if st["bias"] is not None:
        y = y + st["bias"]
    return y.to(_TYPES[case["out"]])


def _plain_rope(st):
    angles, magnitude = _turn_angles(st["case"], st["pos"])
    return _rotate(st["case"], st["x"], angles, magnitude).to(st["x"].dtype)


def _token_rows(st, device):
    """Sequence and place among the sequence's own tokens, for every new token."""
    q, kv = torch.tensor(st["q"], device=device), torch.tensor(st["kv"], device=device)
    seq = torch.repeat_interleave(torch.arange(len(st["q"]), device=device), q)
    i = torch.arange(st["tokens"], device=device) - (torch.cumsum(q, 0) - q)[seq]
    return seq, (kv - q)[seq] + i


def _plain_append(st):
    case = st["case"]
    seq, place = _token_rows(st, "cuda")
    angles, magnitude = _turn_angles(case, place + case["prefix"])
    page = st["pages"][seq, place // case["page"]].long()
    slot = place % case["page"]
    st["k_cache"][page, :, slot] = _rotate(case, st["k_in"], angles, magnitude).to(_TYPES[case["cache"]])
    st["v_cache"][page, :, slot] = st["v_in"].to(_TYPES[case["cache"]])
    return _rotate(case, st["q_in"], angles, magnitude).to(_TYPES[case["dtype"]]), st["k_cache"], st["v_cache"]


def _plain_attention(st):
    case = st["case"]
    hkv, d, page, batch = case["kv_heads"], case["head_dim"], case["page"], case["batch"]
    group, prefix, most = case["heads"] // hkv, case["prefix"], max(st["kv"])
    tokens = st["tokens"]
    q = st["q_in"].float().view(tokens, hkv, group, d) * (1.0 / math.sqrt(d))
    seq, place = _token_rows(st, "cuda")
    # every row against the prefix: [hkv, tokens * group, prefix]
    rows = q.permute(1, 0, 2, 3).reshape(hkv, tokens * group, d)
    pk = st["k_cache"][st["prefix_pages"].long()].permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :prefix].float()
    pv = st["v_cache"][st["prefix_pages"].long()].permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :prefix].float()
    sp = torch.matmul(rows, pk.transpose(1, 2).contiguous())
    # every sequence's rows, padded, against its own keys, padded: [batch, hkv, q_max * group, most]
    own_pages = st["pages"].long()[:, : -(-most // page)]
    ok = st["k_cache"][own_pages].permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)[:, :, :most].float()
    ov = st["v_cache"][own_pages].permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)[:, :, :most].float()
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
        out = out + torch.matmul(pp, pv).view(hkv, tokens, group, d).permute(1, 0, 2, 3)
    y = (out / total[..., None]).reshape(tokens, case["heads"], d)
    return y.to(_TYPES[case["dtype"]]), (top + torch.log(total)).reshape(tokens, case["heads"])


# ------------------------------------------------------------------ the library's operators

def _library(st):
    case, ctx = st["case"], _ctx()
    stream = torch.cuda.current_stream().cuda_stream
    if case["kind"] == "i8":
        m, k, n = case["tokens"], case["in_feat"], case["out_feat"]
        ctx.quantize_i8_device(_tag(case["dtype"]), st["x"].data_ptr(), k, st["xq"].data_ptr(), _up16(k),
                               st["xs"].data_ptr(), m, k, stream)
        ctx.linear_i8_device(st["xq"].data_ptr(), _up16(k), st["xs"].data_ptr(), st["w"].data_ptr(), _up16(k),
                             st["ws"].data_ptr(), None if st["bias"] is None else st["bias"].data_ptr(),
                             _tag(case["out"]), st["y"].data_ptr(), n, m, k, n, stream)
        return st["y"]
    if case["kind"] == "rope":
        x, y = st["x"], st["y"]
        ctx.rope_device(st["rope"], _tag(case["dtype"]), x.data_ptr(), x.stride(0), x.stride(1), y.data_ptr(),
                        y.stride(0), y.stride(1), st["pos"].data_ptr(), case["tokens"], case["heads"],
                        case["head_dim"], stream)
        return y
    q, y = st["q_in"], st["y"]
    if case["kind"] == "append":
        k, v = st["k_in"], st["v_in"]
        ctx.kv_append_device(st["own_cache"], st["own_batch"], st["rope"], _tag(case["dtype"]), st["tokens"],
                             k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), stream,
                             heads=case["heads"], q_ptr=q.data_ptr(), q_token_stride=q.stride(0),
                             q_head_stride=q.stride(1), q_out_ptr=y.data_ptr(), q_out_token_stride=y.stride(0),
                             q_out_head_stride=y.stride(1))
        return y, st["k_cache"], st["v_cache"]
    ctx.attention_device(st["own_cache"], st["own_batch"], _tag(case["dtype"]), st["tokens"], case["heads"],
                         q.data_ptr(), q.stride(0), q.stride(1), y.data_ptr(), y.stride(0), y.stride(1),
                         1.0 / math.sqrt(case["head_dim"]), st["ws"].data_ptr(), st["ws"].numel(), stream,
                         lse_ptr=st["lse"].data_ptr())
    return y, st["lse"]


def run(state):
    if own:
        return _library(state)
    return {"i8": _plain_i8, "rope": _plain_rope, "append": _plain_append,
            "attention": _plain_attention}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ work and exact results

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["kind"] == "i8":
        m, k, n = case["tokens"], case["in_feat"], case["out_feat"]
        return {"bytes": m * k * size[case["dtype"]] + n * k + 4 * n * (2 if case["bias"] else 1)
                + m * n * size[case["out"]], "flops": 2 * m * k * n}
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"] * case["head_dim"]
        return {"bytes": 2 * n * size[case["dtype"]] + 4 * case["tokens"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rot_dim"]}
    q, kv = _lengths(case)
    tokens, d = sum(q), case["head_dim"]
    if case["kind"] == "append":
        cached = tokens * 2 * case["kv_heads"] * d
        return {"bytes": 2 * tokens * case["heads"] * d * size[case["dtype"]] + cached * (size[case["dtype"]]
                + size[case["cache"]]) + 4 * (3 * case["batch"] + 1),
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rot_dim"]}
    keys = sum(n * case["prefix"] + n * (m - n) + n * (n + 1) // 2 for n, m in zip(q, kv))
    cached = (case["prefix"] + sum(kv)) * 2 * case["kv_heads"] * d * size[case["cache"]]
    return {"bytes": cached + 2 * tokens * case["heads"] * d * size[case["dtype"]] + 4 * tokens * case["heads"],
            "flops": 4 * case["heads"] * d * keys}


def _frequency(case, i):
    """Radians a position of pair i, and the magnitude, as plain numbers."""
    r, theta, s = case["rot_dim"], case.get("theta", 10000.0), case.get("factor", 1.0)
    f = theta ** (-2.0 * i / r)
    scaling, original = case.get("scaling", "none"), case.get("original", 4096)
    if scaling == "linear":
        return f / s, 1.0
    if scaling == "bands":
        turns = original * f / (2.0 * math.pi)
        part = min(1.0, max(0.0, (turns - 1.0) / 3.0))
        return f * (part + (1.0 - part) / s), 1.0
    if scaling == "yarn":
        def at(turns):
            return r * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), r - 1)
        part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
        return f * ((1.0 - part) + part / s), 1.0 + 0.1 * math.log(s)
    return f, 1.0


def _exact_rotate(case, x, pos):
    """Complex rotation of x [tokens, heads, head_dim] by pos in 64 bits."""
    r = case["rot_dim"]
    pairs = [_frequency(case, i) for i in range(r // 2)]
    f = torch.tensor([p[0] for p in pairs], dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full((x.shape[0], r // 2), pairs[0][1], dtype=torch.float64, device=x.device),
                       pos.double().unsqueeze(1) * f.unsqueeze(0)).unsqueeze(1)
    x = x.double()
    head = x[..., :r]
    if case["layout"] == "half":
        z = torch.complex(head[..., : r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
        rotated = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], r // 2, 2).contiguous()) * turn
        rotated = torch.view_as_real(z).reshape(head.shape)
    return torch.cat([rotated, x[..., r:]], -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "i8":
        k = case["in_feat"]
        if 2 * case["tokens"] * k * case["out_feat"] > 5e11:
            return None
        x = st["x"].double()
        s = torch.div(x.abs().max(dim=1, keepdim=True).values, 127.0).float().double()
        q = torch.where(s == 0, torch.zeros_like(x), x / torch.where(s == 0, torch.ones_like(s), s)).round()
        y = torch.mm(q, st["w"][:, :k].double().t().contiguous()) * (s * st["ws"].double())
        return y if st["bias"] is None else y + st["bias"].double()
    if case["kind"] == "rope":
        return _exact_rotate(case, st["x"], st["pos"])
    page, prefix = case["page"], case["prefix"]
    begin = [0]
    for n in st["q"]:
        begin.append(begin[-1] + n)
    if case["kind"] == "append":
        pos = torch.cat([torch.arange(m - n, m) for n, m in zip(st["q"], st["kv"])]).cuda() + prefix
        keys, values = _exact_rotate(case, st["k_in"], pos), st["v_in"].double()
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        for b, (n, m) in enumerate(zip(st["q"], st["kv"])):
            j = torch.arange(m - n, m, device="cuda")
            kc[st["pages"][b].long()[j // page], :, j % page] = keys[begin[b]:begin[b + 1]]
            vc[st["pages"][b].long()[j // page], :, j % page] = values[begin[b]:begin[b + 1]]
        return _exact_rotate(case, st["q_in"], pos), kc, vc
    if work(case)["flops"] > 2e12:
        return None
    d, group = case["head_dim"], case["heads"] // case["kv_heads"]
    ys, ls = [], []
    for b, (n, m) in enumerate(zip(st["q"], st["kv"])):
        def sequence(cache):
            """[kv_heads, prefix + m, head_dim]"""
            own_part = cache[st["pages"][b].long()].transpose(0, 1).flatten(1, 2)[:, :m]
            shared = cache[st["prefix_pages"].long()].transpose(0, 1).flatten(1, 2)[:, :prefix]
            return torch.cat([shared, own_part], 1).double()
        q = st["q_in"][begin[b]:begin[b + 1]].double().unflatten(1, (-1, group)).permute(1, 2, 0, 3).flatten(1, 2)
        score = torch.bmm(q, sequence(st["k_cache"]).transpose(1, 2).contiguous()) / math.sqrt(d)
        last = prefix + m - n + torch.arange(n, device="cuda")
        after = torch.arange(prefix + m, device="cuda")[None, :] > last[:, None]
        score = score.unflatten(1, (group, n)).masked_fill(after, -math.inf)
        norm = torch.logsumexp(score, -1)
        weight = torch.exp(score - norm[..., None]).flatten(1, 2)
        y = torch.bmm(weight, sequence(st["v_cache"])).unflatten(1, (group, n))
        ys.append(y.permute(2, 0, 1, 3).reshape(n, case["heads"], d))
        ls.append(norm.permute(2, 0, 1).reshape(n, case["heads"]))
    return torch.cat(ys), torch.cat(ls)
