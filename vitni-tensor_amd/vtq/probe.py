"""ctypes binding of libvtq_probe.so: a measurement helper of bench.py (a
hand-written read-only stream kernel) and the dispatch rules' answers for
tests.  Not part of the quantized-linear boundary."""
from __future__ import annotations

import ctypes
import os

from . import F32, LIB_DIR, Q4_0, Q4_K, Q5_0, Q6_K, Q8_0, REGIME_INTEGER, load_library

_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        load_library()  # torch first, then the HIP libraries: one HIP runtime per process
        path = os.path.join(LIB_DIR, "libvtq_probe.so")
        if not os.path.exists(path):
            raise ImportError(f"{path} is missing (run __graft_entry__.build())")
        L = ctypes.CDLL(path)
        L.vtqp_stream_read.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_void_p,
                                       ctypes.c_void_p]
        L.vtqp_stream_read.restype = ctypes.c_int
        for f in (L.vtqp_canon_form, L.vtqp_kquant_form):
            f.argtypes = [ctypes.c_int] * 4
            f.restype = ctypes.c_int
        vp, sz, i, f = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_float
        L.vtqp_check_quantize_i8.argtypes = [vp, i, vp, sz, vp, sz, vp, sz, sz]
        L.vtqp_check_linear_i8.argtypes = [vp, vp, sz, vp, vp, sz, vp, vp, i, vp, sz, sz, sz, sz]
        L.vtqp_check_rope_call.argtypes = [vp, vp, i, vp, sz, sz, vp, sz, sz, vp, sz, sz, sz]
        L.vtqp_check_append.argtypes = [vp, vp, vp, vp, i, sz, vp, sz, sz, vp, sz, sz, sz, vp, sz, sz, vp, sz, sz]
        L.vtqp_check_attention.argtypes = [vp, vp, vp, i, sz, sz, vp, sz, sz, vp, sz, sz, vp, f]
        L.vtqp_i8_form.argtypes = [i, i, i]
        L.vtqp_attention_plan.argtypes = [vp, vp, i, sz, sz, ctypes.POINTER(i)]
        L.vtqp_own_chunk.argtypes = [i, i, i]
        L.vtqp_slot_of.argtypes = [vp, vp, i, ctypes.c_int64]
        L.vtqp_slot_of.restype = ctypes.c_int64
        _lib = L
    return _lib


# forms of the int8 product, in the library's order
I8_FORMS = ("rows", "slices32", "slices64", "slices128", "tiles128", "pair128", "tiles128x256", "tiles256")


def i8_form(batch: int, in_feat: int, out_feat: int) -> str:
    """The form that vtq_linear_i8_device gives a call."""
    return I8_FORMS[lib().vtqp_i8_form(batch, in_feat, out_feat)]


def refusal(operator: str, *args):
    """(status, text) that a serving operator's call with these arguments (without context, workspace and
    stream) gets before anything is launched; no GPU is needed."""
    text = ctypes.c_char_p()
    rc = getattr(lib(), "vtqp_check_" + operator)(ctypes.byref(text), *args)
    return rc, (text.value or b"").decode()


PLAN = ("group", "page_shift", "prefix_rows", "prefix_splits", "prefix_chunk", "own_rows", "own_splits", "own_grain",
        "shared_prefix", "shared_own", "prefix_per_xcd", "own_per_xcd")


def attention_plan(cache, batch, ggml_type, tokens, heads):
    """How vtq_attention_device splits a call (AttentionPlan of vtq_attention_plan.h); None where it is refused."""
    out = (ctypes.c_int * len(PLAN))()
    rc = lib().vtqp_attention_plan(cache.ref, batch.ref, ggml_type, tokens, heads, out)
    return None if rc else dict(zip(PLAN, out))


def own_chunk(keys, splits, grain):
    """Keys to each range of a sequence's own."""
    return lib().vtqp_own_chunk(keys, splits, grain)


def stream_read(ptr: int, nbytes: int, workgroups: int, sink_ptr: int, stream: int) -> None:
    """Launch a read-only stream of `nbytes` (a multiple of 16) at device
    address `ptr` with `workgroups` workgroups of 256 threads on `stream`."""
    rc = lib().vtqp_stream_read(ptr, nbytes, workgroups, sink_ptr, stream)
    if rc != 0:
        raise RuntimeError(f"vtqp_stream_read: hipError {rc}")


GEMV, LDS_OPERAND, PER_WAVE = 0, 1, 2  # besides split-K: 300 + piece, 600 + piece with two token tiles to a wave


def form(ggml_type: int, regime: int, batch: int, in_feat: int, out_feat: int) -> int:
    """The kernel form that a call takes: GEMV (one slice per batch row); for
    integer Q4_K and Q6_K LDS_OPERAND, PER_WAVE or split-K's number; else, for
    the pinned dot over a batch, 10 * token tiles of a wave + waves to a tile."""
    if ggml_type == Q6_K or (ggml_type == Q4_K and regime == REGIME_INTEGER):
        return lib().vtqp_kquant_form(ggml_type, batch, in_feat, out_feat)
    fmt = {Q8_0: 0, Q5_0: 1, Q4_0: 2, F32: 3, Q4_K: 4}[ggml_type]
    return lib().vtqp_canon_form(fmt, batch, in_feat, out_feat)
