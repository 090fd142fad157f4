"""Checks on the gfx950 code of the serving kernels that load straight to LDS.

load_to_lds sets m0, the LDS base of `buffer_load ... lds`, inside inline asm; m0 is a
reserved register that the compiler does not save around an asm statement, so no
instruction of its own may use it in these kernels.  CPU only (hipcc cross-compiles)."""
import os
import re
import shutil
import subprocess

import pytest

from test_asm_checks import FLAGS, HIPCC, ROOT, _functions, _scratch_sizes

CSRC = os.path.join(ROOT, "vitni-tensor_amd", "csrc")


@pytest.fixture(scope="module", params=["cache_attention.hip", "i8_linear.hip"])
def asm(request, tmp_path_factory):
    if not (os.path.exists(HIPCC) or shutil.which("hipcc")):
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm") / "out.s"
    subprocess.run([HIPCC if os.path.exists(HIPCC) else "hipcc", *FLAGS, "--cuda-device-only", "-S", "-o", str(out),
                    os.path.join(CSRC, request.param)], check=True, stdout=subprocess.DEVNULL,
                   stderr=subprocess.DEVNULL, timeout=900)
    return request.param, _functions(out.read_text())


def test_m0_is_set_only_for_the_loads_to_lds(asm):
    name, functions = asm
    loads = 0
    for kernel, body in functions.items():
        code = [l for l in body if l and not l.startswith((";", "."))]
        for i, line in enumerate(code):
            if "lds" in line.split() and line.startswith("buffer_load"):
                loads += 1
            if not re.search(r"\bm0\b", line):
                continue
            # the asm's own three: s_mov_b32 m0, sN ; s_nop 0 ; buffer_load_dwordx4 ... lds
            assert re.match(r"s_mov_b32 m0, s\d+$", line), (kernel, line)
            assert code[i + 1] == "s_nop 0", (kernel, code[i + 1])
            assert re.match(r"buffer_load_dwordx4 v\d+, s\[\d+:\d+\], 0 offen lds$", code[i + 2]), (kernel, code[i + 2])
    assert loads > 20, name


def test_loops_of_the_16_bit_attention_wait_only_for_their_own_loads(asm):
    # A wait for every load in flight inside a tile's loop would undo the loads ahead: the
    # compiler puts one before the use of an ordinary load's result.  In the loops (blocks
    # with products and loads to LDS) of heads of up to 128 elements none may stand beside
    # the kernel's own, which follow a barrier's place.
    name, functions = asm
    if name != "cache_attention.hip":
        pytest.skip("attention only")
    checked = 0
    for kernel, body in functions.items():
        if not re.search(r"attention_kernelI(DF16_DF16_|DF16bDF16b)Li(64|128)", kernel):
            continue
        checked += 1
        code = [l for l in body if l and not l.startswith(";")]
        for i, line in enumerate(code):
            if line.startswith("v_readlane_b32") and i and re.match(r"s_waitcnt vmcnt\(0\)", code[i - 1]):
                raise AssertionError((kernel, code[i - 3:i + 1]))
    assert checked == 4


def test_int8_kernels_do_not_spill():
    if not (os.path.exists(HIPCC) or shutil.which("hipcc")):
        pytest.skip("hipcc not available")
    sizes = _scratch_sizes(os.path.join(CSRC, "i8_linear.hip"))
    kernels = {k: v for k, v in sizes.items() if "kernel" in k}
    assert kernels and not {k: v for k, v in kernels.items() if v}
