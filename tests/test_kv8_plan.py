"""How an attention call over an 8-bit cache is split, and the gfx950 code of the kernels of 8-bit caches, beams and
pages, both without a GPU (hipcc cross-compiles)."""
import os
import random
import re
import shutil
import subprocess

import pytest

import vtq
from test_asm_checks import FLAGS, HIPCC, ROOT, _functions
from vtq import probe

A = 1 << 20  # an aligned address; nothing is read
CSRC = os.path.join(ROOT, "vitni-tensor_amd", "csrc")
SOURCES = ("kv8_append.hip", "kv8_attention.hip", "beam_select.hip", "cache_pages.hip")


def _check(ggml_type, kv_heads, group, head_dim, page, batch, max_q, max_len, max_pages, prefix, tokens):
    heads = kv_heads * group
    cache = vtq.Kv8Cache(A, A, A, A, 1 << 20, page, kv_heads, head_dim)
    desc = vtq.KvBatch(batch, A, A, A, max_pages, max_q=max_q, max_len=max_len, prefix_len=prefix, prefix_pages=A)
    p = probe.attention_plan(cache, desc, ggml_type, tokens, heads)
    need = vtq.load_library().vtq_kv8_attention_workspace(cache.ref, desc.ref, ggml_type, tokens, heads)
    if p is None:
        assert need == 0
        return None
    halves = 2 if head_dim > 128 else 1
    parts = p["prefix_splits"] + p["own_splits"]
    assert p["group"] == group and 1 << p["page_shift"] == page
    assert p["own_splits"] >= 1 and halves <= parts <= 128  # two workgroups to a row never write y themselves
    # the prefix has workgroups, or short ones stand inside those of prompts that fill the chip
    inside = prefix > 0 and p["prefix_splits"] == 0
    assert not inside or (prefix <= 4096 and p["shared_own"] and parts == halves)
    assert (p["prefix_splits"] >= 1) == (prefix > 0 and not inside)
    assert need >= (parts * tokens * heads * (4 * head_dim + 8) if parts > 1 else 0)
    if prefix and not inside:
        assert p["prefix_chunk"] % 32 == 0
        assert (p["prefix_splits"] - 1) * p["prefix_chunk"] < prefix <= p["prefix_splits"] * p["prefix_chunk"]
        assert p["prefix_rows"] * 32 * (4 if p["shared_prefix"] else 1) >= tokens * group
    for keys in (0, 1, 31, 33, 129, 1000, max_pages * page // 2 + 1, max_pages * page):
        if keys <= max_pages * page:
            chunk = probe.own_chunk(keys, p["own_splits"], p["own_grain"])
            assert chunk % 32 == 0 and chunk * p["own_splits"] >= keys
    assert p["own_rows"] >= 1 and (inside or p["shared_prefix"] == (tokens * group > 32))
    assert 8 * p["prefix_per_xcd"] >= halves * kv_heads * p["prefix_splits"] * p["prefix_rows"]
    assert 8 * p["own_per_xcd"] >= halves * kv_heads * p["own_splits"] * batch * p["own_rows"]
    # as the kernel takes them: every row tile of every range of keys once
    for units, rows, per in ((kv_heads * p["prefix_splits"], halves * p["prefix_rows"], p["prefix_per_xcd"]),
                             (kv_heads * p["own_splits"] * batch, halves * p["own_rows"], p["own_per_xcd"])):
        if units * rows > 2000 or not units:
            continue
        turns, last = units // 8, units % 8
        share = 8 // last if last else 1
        seen = []
        for xcd in range(8):
            for mine in range(per):
                if mine < turns * rows:
                    seen.append((mine // rows * 8 + xcd, mine % rows))
                elif xcd < last * share and (mine - turns * rows) * share + xcd // last < rows:
                    seen.append((turns * 8 + xcd % last, (mine - turns * rows) * share + xcd // last))
        assert sorted(seen) == [(u, t) for u in range(units) for t in range(rows)]
    assert p["prefix_per_xcd"] >= 0 and 8 * (p["prefix_per_xcd"] + p["own_per_xcd"]) * 256 < 1 << 32
    return p


@pytest.mark.parametrize("ggml_type", [vtq.F32, vtq.F16, vtq.BF16])
@pytest.mark.parametrize("kv_heads", [1, 2, 3, 4, 8, 65535])
def test_plans_cover_the_work(ggml_type, kv_heads):
    rng = random.Random(17 * kv_heads + ggml_type)

    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    planned = 0
    for _ in range(400):
        page = rng.choice([16, 64, 256, 4096])
        batch, max_q = log(1, 4096), rng.choice([0, 1, 1, log(2, 8192)])
        group = rng.choice([1, 1, 4, 7, 8, 64]) if kv_heads < 65535 else 1
        own = max(max_q, log(1, 1 << 20))
        prefix = rng.choice([0, log(1, 1 << 20), log(1, 40)])
        tokens = max(1, min(rng.choice([batch * max(1, max_q), log(1, 10000)]), (1 << 25) // (kv_heads * group)))
        planned += _check(ggml_type, kv_heads, group, rng.choice([16, 64, 80, 128, 144, 256]), page, batch, max_q,
                          rng.choice([0, 0, own, 1]), rng.choice([-(-own // page), 0]), prefix, tokens) is not None
    assert planned > 10  # the others are refused


@pytest.mark.parametrize("ggml_type", [vtq.F32, vtq.F16, vtq.BF16])
def test_plans_of_the_largest_calls(ggml_type):
    for head_dim, most in ((128, 22), (256, 20)):
        for args in ((1, 8, head_dim, 16, 1, 8192, 0, 512, 0, 8192), (3, 8, head_dim, 16, 1, 500, 0, 32, 0, 500),
                     (4, 8, head_dim, 16, 1, 1000, 0, 64, 0, 1000), (2, 16, head_dim, 16, 1, 333, 0, 64, 70, 333),
                     (1, 8, head_dim, 16, 1, 1 << (most - 3), 0, (1 << 30) // 16 - 1, (1 << 30) - 1, 1 << (most - 3)),
                     (8, 1, head_dim, 16, 1 << (most - 3), 1, 0, 4, 7, 1 << (most - 3)),
                     (8, 1, head_dim, 16, 1 << (most - 3), 1, 0, 4, 0, 1 << (most - 3)),
                     (1, 4, head_dim, 16, 1, 1 << 20, 0, 1 << 16, 1 << 20, 1 << 20)):
            assert _check(ggml_type, *args), args
        # one workgroup more
        assert _check(ggml_type, 8, 1, head_dim, 16, (1 << (most - 3)) + 1, 1, 0, 4, 7, (1 << (most - 3)) + 1) is None


def test_no_source_reads_the_environment():
    for name in SOURCES + ("vtq_rope.h", "vtq_attention_rows.h"):
        with open(os.path.join(CSRC, name)) as f:
            assert "getenv" not in f.read(), name


@pytest.fixture(scope="module", params=SOURCES)
def asm(request, tmp_path_factory):
    if not (os.path.exists(HIPCC) or shutil.which("hipcc")):
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm") / "out.s"
    subprocess.run([HIPCC if os.path.exists(HIPCC) else "hipcc", *FLAGS, "--cuda-device-only", "-S", "-o", str(out),
                    os.path.join(CSRC, request.param)], check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL,
                   timeout=900)
    return request.param, out.read_text()


def test_m0_is_set_only_for_the_loads_to_lds(asm):
    name, text = asm
    loads = 0
    for kernel, body in _functions(text).items():
        code = [l for l in body if l and not l.startswith((";", "."))]
        has_loads = any(l.startswith("buffer_load") and "lds" in l.split() for l in code)
        for i, line in enumerate(code):
            if not (has_loads and re.search(r"\bm0\b", line)):
                continue
            loads += 1
            assert re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)$", line), (kernel, line)
            assert code[i + 1] == "s_nop 0", (kernel, code[i + 1])
            assert re.match(r"buffer_load_dwordx4 v\d+, s\[\d+:\d+\], 0 offen lds$", code[i + 2]), (kernel, code[i + 2])
    assert (loads > 20) == (name == "kv8_attention.hip")


def test_scratch_memory_and_the_dispatch_packet(asm):
    # Scratch accesses share a counter with the tiles' loads; an array that the compiler puts in LDS has its size read
    # from the dispatch packet, in host memory, at 13 us a launch.
    name, text = asm
    sizes, packet, current = {}, {}, None
    for line in text.split("\n"):
        m = re.match(r"^([_A-Za-z][\w.$]*):", line)
        current = m.group(1) if m and not line.startswith(".L") else current
        m = re.match(r"^; ScratchSize: (\d+)", line.strip())
        if m:
            sizes[current] = int(m.group(1))
        m = re.match(r"\.amdhsa_user_sgpr_dispatch_ptr (\d)", line.strip())
        if m:
            packet[current] = int(m.group(1))
    kernels = [k for k in sizes if "kernel" in k]
    assert len(kernels) >= 3 and len(packet) >= 3
    assert not any(packet.values()), packet
    assert not {k: sizes[k] for k in kernels if sizes[k]}


def test_no_wait_for_all_loads_stands_beside_products(asm):
    # the tiles ahead load to LDS, which the compiler does not count: a wait of its own for an ordinary load inside a
    # loop would be one for all of them
    name, text = asm
    if name != "kv8_attention.hip":
        pytest.skip("attention only")
    blocks = 0
    for kernel, body in _functions(text).items():
        block = []
        for line in body + [".LBB"]:
            if not line.startswith(".LBB"):
                block.append(line)
                continue
            if sum(l.startswith("v_mfma") for l in block) >= 4:
                blocks += 1
                assert not [l for l in block if re.match(r"s_waitcnt.*vmcnt\(0\)", l)], kernel
            block = []
    assert blocks >= 18 * 3
