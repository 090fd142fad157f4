"""Which attention calls over an 8-bit cache give the shared prefix to the sequences' own workgroups, asked without a
GPU: only such as fill the chip with rows, or whose prefix is short."""
import random

import pytest

import vtq
from vtq import probe

A = 1 << 20  # an aligned address; nothing is read


def _plan(ggml_type, q_lens, own, prefix, heads, kv_heads, head_dim, page=16, tokens=None, max_q=None):
    cache = vtq.Kv8Cache(A, A, A, A, 1 << 20, page, kv_heads, head_dim)
    desc = vtq.KvBatch(len(q_lens), A, A, A, -(-own // page), max_q=max(q_lens) if max_q is None else max_q,
                       prefix_len=prefix, prefix_pages=A)
    return probe.attention_plan(cache, desc, ggml_type, sum(q_lens) if tokens is None else tokens, heads)


# each measured the slower with the prefix inside, most by far
@pytest.mark.parametrize("ggml_type,q_lens,own,prefix,heads,kv_heads,head_dim", [
    # fewer workgroups than the chip takes, each through all of the prefix
    (vtq.BF16, [60], 64, 4096, 32, 8, 128), (vtq.BF16, [60], 64, 1000, 32, 8, 128), (vtq.BF16, [60], 64, 161, 32, 8, 128),
    (vtq.BF16, [100], 100, 4096, 32, 8, 128), (vtq.BF16, [60] * 2, 64, 4000, 32, 8, 128),
    (vtq.BF16, [16] * 8, 100, 4096, 32, 8, 128), (vtq.BF16, [6] * 16, 100, 4000, 64, 8, 128),
    (vtq.F32, [60], 64, 4096, 32, 8, 128), (vtq.F16, [400], 400, 4096, 32, 8, 128),
    # tiles of 128 rows with a few in each
    (vtq.BF16, [9] * 64, 100, 4096, 32, 8, 128), (vtq.BF16, [9] * 64, 100, 1000, 32, 8, 128),
    # decoding sequences beside one chunk of a prompt
    (vtq.BF16, [1] * 63 + [512], 900, 2000, 32, 8, 128), (vtq.BF16, [1] * 63 + [512], 900, 300, 32, 8, 128),
    (vtq.F16, [1] * 20 + [512], 900, 300, 32, 8, 128), (vtq.F32, [1] * 63 + [512], 900, 40, 32, 8, 128),
    # heads whose rows are joined anyway
    (vtq.F16, [64] * 62, 64, 200, 8, 4, 256), (vtq.BF16, [1024], 1024, 1000, 32, 32, 256)])
def test_prefixes_with_workgroups_of_their_own(ggml_type, q_lens, own, prefix, heads, kv_heads, head_dim):
    p = _plan(ggml_type, q_lens, own, prefix, heads, kv_heads, head_dim)
    assert p["prefix_splits"] >= 1


def test_a_long_prefix_has_enough_workgroups():
    # 4096 keys and one more differ little
    for q_lens, own in (([60], 64), ([100], 100), ([60] * 2, 64), ([16] * 8, 100)):
        for prefix in (4096, 4097):
            p = _plan(vtq.BF16, q_lens, own, prefix, 32, 8, 128)
            assert 8 * (p["prefix_per_xcd"] + p["own_per_xcd"]) >= 128, (q_lens, prefix)


@pytest.mark.parametrize("ggml_type,q_lens,own,prefix,heads,kv_heads,head_dim", [
    (vtq.BF16, [164] * 12, 218, 161, 32, 8, 96), (vtq.BF16, [164] * 12, 218, 2000, 32, 8, 96),
    (vtq.BF16, [2048], 2048, 161, 32, 8, 128), (vtq.BF16, [2048], 2048, 4096, 32, 8, 128),
    (vtq.F16, [1000] * 4, 1000, 1000, 32, 8, 64), (vtq.BF16, [9] * 64, 100, 161, 32, 8, 128),
    (vtq.BF16, [129] * 117, 172, 1000, 8, 2, 64), (vtq.BF16, [100] * 40, 100, 2000, 64, 64, 128)])
def test_prefixes_inside_prompts(ggml_type, q_lens, own, prefix, heads, kv_heads, head_dim):
    assert _plan(ggml_type, q_lens, own, prefix, heads, kv_heads, head_dim)["prefix_splits"] == 0


def test_what_is_inside_fills_the_chip_or_is_short():
    rng = random.Random(11)

    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    inside = 0
    for _ in range(6000):
        kv_heads, group = rng.choice([1, 2, 4, 8, 8, 32]), rng.choice([1, 4, 7, 8])
        head_dim = rng.choice([64, 96, 128, 128, 256])
        batch, max_q = log(1, 200), log(8, 3000)
        tokens = min(rng.choice([batch * max_q, rng.randint(max_q, batch * max_q)]), 20000)
        prefix = log(1, 8192)
        p = _plan(rng.choice([vtq.F32, vtq.F16, vtq.BF16]), [max_q] * batch, max_q + log(1, 300), prefix, kv_heads * group,
                  kv_heads, head_dim, tokens=tokens)
        if p is None or p["prefix_splits"]:
            continue
        inside += 1
        tiles = p["own_rows"] * batch
        assert 128 * tiles <= 5 * tokens * group  # tiles have rows
        with_rows = kv_heads * (2 if head_dim > 128 else 1) * min(tiles, tokens * group / 128 + batch)
        assert prefix <= (512 if with_rows <= 64 else 1024 if with_rows <= 128 else 4096)
        assert head_dim <= 128 or prefix <= 64
    assert inside > 500
