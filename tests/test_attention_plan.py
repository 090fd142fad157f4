"""How an attention call's work is split, asked without a GPU."""
import os
import random
import subprocess
import sys

import pytest

import vtq
from vtq import probe

A = 1 << 20  # an aligned address; nothing is read

_WORKSPACES = f"""
import sys
sys.path.insert(0, {os.path.dirname(os.path.dirname(os.path.abspath(vtq.__file__)))!r})
import vtq
A = {A}
for batch, max_q, own, prefix in ((4, 1, 1000, 0), (512, 1, 300, 32768), (1, 2048, 2048, 0), (16, 6, 4000, 1003)):
    cache = vtq.KvCache(vtq.BF16, A, A, 1 << 20, 16, 8, 128)
    desc = vtq.KvBatch(batch, A, A, A, -(-own // 16), max_q=max_q, prefix_len=prefix, prefix_pages=A)
    lib = vtq.load_library()
    print(lib.vtq_attention_workspace(cache.ref, desc.ref, vtq.BF16, batch * max_q, 32))
"""


@pytest.mark.parametrize("value", ["0", "200", "-3", "x"])
def test_the_environment_does_not_reach_the_plan(value):
    env = {k: v for k, v in os.environ.items() if k != "OWNS"}

    def sizes(**more):
        return subprocess.run([sys.executable, "-c", _WORKSPACES], env={**env, **more}, check=True, capture_output=True,
                              text=True, timeout=300).stdout.split()

    plain = sizes()
    assert len(plain) == 4 and int(plain[0]) > 0
    assert sizes(OWNS=value) == plain


def test_no_serving_source_reads_the_environment():
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(vtq.__file__))), "csrc")
    for name in ("cache_attention.hip", "i8_linear.hip", "rope_kv.hip", "vtq_serve_api.hip", "vtq_serve.h",
                 "vtq_serve_checks.h", "vtq_i8_rules.h", "vtq_attention_plan.h", "vtq_lds_load.h"):
        with open(os.path.join(csrc, name)) as f:
            assert "getenv" not in f.read(), name


def _up(x, y):
    return -(-x // y)


def _check(ggml_type, cache_type, kv_heads, group, head_dim, page, batch, max_q, max_len, max_pages, prefix, tokens):
    heads = kv_heads * group
    cache = vtq.KvCache(cache_type, A, A, 1 << 20, page, kv_heads, head_dim)
    desc = vtq.KvBatch(batch, A, A, A, max_pages, max_q=max_q, max_len=max_len, prefix_len=prefix, prefix_pages=A)
    p = probe.attention_plan(cache, desc, ggml_type, tokens, heads)
    need = vtq.load_library().vtq_attention_workspace(cache.ref, desc.ref, ggml_type, tokens, heads)
    if p is None:
        assert need == 0
        return None
    assert p["group"] == group and 1 << p["page_shift"] == page
    # at least one own range, no more parts than the join takes, and a workspace that holds them
    parts = p["prefix_splits"] + p["own_splits"]
    assert p["own_splits"] >= 1 and parts <= 128
    assert (p["prefix_splits"] >= 1) == (prefix > 0)
    assert need >= (parts * tokens * heads * (4 * head_dim + 8) if parts > 1 else 0)
    # the prefix's ranges: every key in one of them, none of them empty, whole tiles
    if prefix:
        assert p["prefix_chunk"] % (32 if p["shared_prefix"] else 128) == 0
        assert (p["prefix_splits"] - 1) * p["prefix_chunk"] < prefix <= p["prefix_splits"] * p["prefix_chunk"]
    # a sequence's own, whatever its length turns out to be
    assert p["own_grain"] in ((32, 128) if p["shared_own"] else (128,))
    for keys in (0, 1, 31, 33, 129, 1000, max_pages * page // 2 + 1, max_pages * page):
        if keys <= max_pages * page:
            chunk = probe.own_chunk(keys, p["own_splits"], p["own_grain"])
            assert chunk % p["own_grain"] == 0 and chunk * p["own_splits"] >= keys
    # row tiles: all rows of the prefix; some of a sequence's, whose workgroups take several
    waves = 2 if 32 * (64 if head_dim <= 64 else 128 if head_dim <= 128 else 256) * (
        4 if cache_type == vtq.F32 else 2) > 16384 else 4
    assert p["shared_prefix"] == (tokens * group > 32)
    if prefix:
        assert p["prefix_rows"] * 32 * (waves if p["shared_prefix"] else 1) >= tokens * group
    assert p["own_rows"] >= 1
    # the grid: a workgroup to every part of the work, and fewer than 2^32 threads
    assert 8 * p["prefix_per_xcd"] >= kv_heads * p["prefix_splits"] * p["prefix_rows"]
    assert 8 * p["own_per_xcd"] >= kv_heads * p["own_splits"] * batch * p["own_rows"]
    assert p["prefix_per_xcd"] >= 0 and 8 * (p["prefix_per_xcd"] + p["own_per_xcd"]) * waves * 64 < 1 << 32
    return p


PAIRS = [(vtq.F32, vtq.F32), (vtq.F16, vtq.F16), (vtq.BF16, vtq.BF16), (vtq.F32, vtq.F16), (vtq.F32, vtq.BF16)]


@pytest.mark.parametrize("ggml_type,cache_type", PAIRS)
@pytest.mark.parametrize("kv_heads", [1, 2, 3, 4, 8, 65535])
def test_plans_cover_the_work(ggml_type, cache_type, kv_heads):
    rng = random.Random(17 * kv_heads + 3 * ggml_type + cache_type)

    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    planned = 0
    for _ in range(400):
        page = rng.choice([8, 16, 64, 256, 4096])
        batch, max_q = log(1, 4096), rng.choice([0, 1, 1, log(2, 8192)])
        group = rng.choice([1, 1, 4, 7, 8, 64]) if kv_heads < 65535 else 1
        own = max(max_q, log(1, 1 << 20))
        prefix = rng.choice([0, log(1, 1 << 20), log(1, 40)])
        tokens = max(1, min(rng.choice([batch * max(1, max_q), log(1, 10000)]), (1 << 25) // (kv_heads * group)))
        planned += _check(ggml_type, cache_type, kv_heads, group, rng.choice([8, 64, 80, 128, 256]), page, batch, max_q,
                          rng.choice([0, 0, own, 1]), rng.choice([_up(own, page), 0]), prefix, tokens) is not None
    assert planned > 20  # the others are refused


@pytest.mark.parametrize("ggml_type,cache_type", PAIRS)
def test_plans_of_prompts_and_of_the_largest_calls(ggml_type, cache_type):
    for args in ((4, 8, 64, 16, 1, 2048, 0, 128, 0, 2048), (2, 16, 128, 16, 1, 4096, 0, 256, 0, 4096),
                 (1, 8, 128, 64, 1, 8192, 0, 128, 0, 8192), (1, 4, 64, 16, 9, 500, 0, 32, 1000, 4500),
                 (1, 8, 128, 16, 1, 1 << 22, 0, (1 << 30) // 16 - 1, (1 << 30) - 1, 1 << 22),
                 (1, 4, 256, 8, 1, 1 << 23, 0, 1 << 20, 1 << 20, 1 << 23),
                 (65535, 1, 64, 8, 32, 1, 0, 4, 1 << 20, 32), (8, 1, 64, 16, 1 << 18, 1, 0, 4, 7, 1 << 18)):
        assert _check(ggml_type, cache_type, *args), args
