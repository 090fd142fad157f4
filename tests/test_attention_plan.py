"""How an attention call's work is split, asked without a GPU."""
import os
import subprocess
import sys

import pytest

import vtq

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
                 "vtq_serve_checks.h", "vtq_i8_rules.h", "vtq_lds_load.h"):
        with open(os.path.join(csrc, name)) as f:
            assert "getenv" not in f.read(), name
