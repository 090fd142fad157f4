"""Where the attention kernels' gfx950 code touches scratch memory.  Loads to LDS and scratch memory share one counter
of loads in flight, so a spilled register read back among a tile's products waits for the tiles loading ahead.  CPU
only (hipcc cross-compiles)."""
import os
import re
import shutil
import subprocess

import pytest

from test_asm_checks import FLAGS, HIPCC, ROOT, _functions

SOURCE = os.path.join(ROOT, "vitni-tensor_amd", "csrc", "cache_attention.hip")
TYPES = {"f": "f32", "DF16_": "f16", "DF16b": "bf16"}
# bytes a lane at most.  Heads of up to 256 elements keep sums of 8 x 16 registers and a query of 64 or more, and
# spill inside the loops too: known, and no more than this.
SCRATCH = {("f16", 128): 16, ("bf16", 128): 16, ("f16", 256): 176, ("bf16", 256): 176, ("f32", 256): 512}


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not (os.path.exists(HIPCC) or shutil.which("hipcc")):
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm") / "out.s"
    subprocess.run([HIPCC if os.path.exists(HIPCC) else "hipcc", *FLAGS, "--cuda-device-only", "-S", "-o", str(out),
                    SOURCE], check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL, timeout=900)
    text, sizes, current = out.read_text(), {}, None
    for line in text.split("\n"):
        m = re.match(r"^([_A-Za-z][\w.$]*):", line)
        current = m.group(1) if m and not line.startswith(".L") else current
        m = re.match(r"^; ScratchSize: (\d+)", line.strip())
        if m:
            sizes[current] = int(m.group(1))
    found = {}
    for symbol, body in _functions(text).items():
        m = re.search(r"attention_kernelI(f|DF16_|DF16b)(f|DF16_|DF16b|S\d*_)Li(\d+)", symbol)
        if m:
            found[TYPES[m.group(1)], m.group(2), int(m.group(3))] = sizes[symbol], body
    assert len(found) == 15  # five pairs of types, three sizes
    return found


def test_scratch_memory_of_every_kernel(kernels):
    for (q, cache, d), (size, _) in kernels.items():
        assert size <= SCRATCH.get((q, d), 0), (q, cache, d, size)


def test_products_of_up_to_128_elements_stand_beside_no_scratch_access(kernels):
    for (q, cache, d), (_, body) in kernels.items():
        if d > 128:
            continue
        blocks, products = [[]], 0
        for line in body:
            if re.match(r"\.LBB|s_c?branch", line):
                blocks.append([])
            blocks[-1].append(line)
        for block in blocks:
            if not any(line.startswith("v_mfma") for line in block):
                continue
            products += 1
            bad = [line for line in block if line.startswith("scratch_") or "vmcnt(0)" in line]
            assert not bad, (q, cache, d, block[0], bad)
        assert products >= 6, (q, cache, d)
