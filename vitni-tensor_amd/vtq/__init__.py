"""vtq -- Python host mirror of vitni-tensor's quantized linear API over libvtq.

The functions keep the reference's names, argument meaning and error
behaviour (src/ops/quant.rs, src/model/forward_quantized.rs:663-785):
``x`` is ``[batch, in_feat]`` float32, ``w`` the GGUF block bytes of
``W[out_feat, in_feat]``, ``y_out`` ``[batch, out_feat]`` float32 written in
place.  A failing call raises the exception that mirrors the reference's
``Error`` variant (src/error.rs:7-63) with the reference's message.

All compute runs in libvtq on the GPU.  If libvtq.so is missing or no GPU is
present the calls raise; there is no CPU fallback in this package.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_DIR = os.path.join(os.path.dirname(_HERE), "lib")
LIB_PATH = os.path.join(LIB_DIR, "libvtq.so")

# GGUF tensor type tags (src/model/gguf.rs:127-139)
F32, F16, Q4_0, Q5_0, Q8_0, Q4_K, Q6_K = 0, 1, 2, 6, 8, 12, 14
BF16 = 30  # activations and caches of the serving operators only
TYPE_NAMES = {F32: "F32", F16: "F16", Q4_0: "Q4_0", Q5_0: "Q5_0", Q8_0: "Q8_0", Q4_K: "Q4_K", Q6_K: "Q6_K",
              BF16: "BF16"}
BLOCK = {Q4_0: (32, 18), Q5_0: (32, 22), Q8_0: (32, 34), Q4_K: (256, 144), Q6_K: (256, 210)}

REGIME_INTEGER = 0       # std-parallel build: integer Q4_K
REGIME_FLOAT_FUSED = 1   # default build: float-fused Q4_K

# rotary layouts and scalings of long contexts (include/vtq.h)
ROPE_INTERLEAVED, ROPE_HALF = 0, 1
ROPE_SCALE_NONE, ROPE_SCALE_LINEAR, ROPE_SCALE_BANDS, ROPE_SCALE_YARN = 0, 1, 2, 3

OK, E_INTERNAL, E_GPU, E_NOT_IMPLEMENTED, E_INVALID_ARGUMENT = 0, 1, 2, 3, 4
E_MALFORMED, E_TRUNCATED, E_OVERFLOW, E_SHAPE_MISMATCH, E_INVALID_SHAPE = 5, 6, 7, 8, 9


class VtqError(Exception):
    """Base of the mirrored vitni_tensor::error::Error variants."""

    code = -1

    def __init__(self, message: str):
        super().__init__(message)
        self.message = message


class Internal(VtqError):
    """Error::Internal(&'static str) -- shape and length violations."""

    code = E_INTERNAL


class GpuError(VtqError):
    """Error::GpuError -- a HIP call failed."""

    code = E_GPU


class NotImplementedDtype(VtqError):
    """Error::NotImplemented -- dtype (or size) not supported."""

    code = E_NOT_IMPLEMENTED


class InvalidArgument(VtqError):
    """Null pointer / context misuse (ruled out by Rust's types in the reference)."""

    code = E_INVALID_ARGUMENT


class Malformed(VtqError):
    """Error::Malformed -- a GGUF file that violates the format."""

    code = E_MALFORMED


class Truncated(VtqError):
    """Error::Truncated -- a GGUF file that ends before a field."""

    code = E_TRUNCATED


class Overflow(VtqError):
    """Error::Overflow -- a GGUF length or offset whose arithmetic overflows."""

    code = E_OVERFLOW


class ShapeMismatch(VtqError):
    """Error::ShapeMismatch -- a norm weight whose length is not the model dimension."""

    code = E_SHAPE_MISMATCH


class InvalidShape(VtqError):
    """Error::InvalidShape -- an empty prompt, or prompt + new tokens past seq_len."""

    code = E_INVALID_SHAPE


_ERRORS = {c.code: c for c in (Internal, GpuError, NotImplementedDtype, InvalidArgument, Malformed, Truncated,
                               Overflow, ShapeMismatch, InvalidShape)}


def error_class(code: int):
    """The exception class of a libvtq / libvtq_runtime status code."""
    return _ERRORS.get(code, GpuError)

_lib: Optional[ctypes.CDLL] = None


def load_library(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load libvtq.so (built in-tree by ``make -C vitni-tensor_amd``)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise ImportError(f"libvtq.so not built: {path} is missing (run __graft_entry__.build())")
    # One HIP runtime per process: torch's ROCm wheel loads its own
    # libamdhip64 (NEEDED "libamdhip64.so", SONAME libamdhip64.so.7).  Loading
    # torch first lets libvtq's NEEDED libamdhip64.so.7 resolve to that same
    # copy by SONAME; the other order would map a second runtime into the
    # process and the second one would find no device.
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    lib = ctypes.CDLL(path)
    vp, sz, i = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int
    lib.vtq_create.argtypes = [i, ctypes.POINTER(vp)]
    lib.vtq_create.restype = i
    lib.vtq_destroy.argtypes = [vp]
    lib.vtq_destroy.restype = None
    lib.vtq_last_error.argtypes = [vp]
    lib.vtq_last_error.restype = ctypes.c_char_p
    lib.vtq_version.argtypes = []
    lib.vtq_version.restype = ctypes.c_char_p
    host_sig = [vp, vp, sz, vp, sz, vp, sz, sz, sz, sz]
    for name in ("vtq_linear_q4_k_integer", "vtq_linear_q6_k_integer", "vtq_linear_q4_k_fused", "vtq_linear_q4_0"):
        f = getattr(lib, name)
        f.argtypes = host_sig
        f.restype = i
    lib.vtq_linear.argtypes = [vp, i, i, vp, sz, vp, sz, vp, sz, sz, sz, sz]
    lib.vtq_linear.restype = i
    lib.vtq_release_weights.argtypes = [vp, vp]
    lib.vtq_release_weights.restype = i
    lib.vtq_linear_device.argtypes = [vp, i, i, vp, vp, sz, vp, sz, sz, sz, vp]
    lib.vtq_linear_device.restype = i
    lib.vtq_quantize_i8_device.argtypes = [vp, i, vp, sz, vp, sz, vp, sz, sz, vp]
    lib.vtq_quantize_i8_device.restype = i
    lib.vtq_linear_i8_device.argtypes = [vp, vp, sz, vp, vp, sz, vp, vp, i, vp, sz, sz, sz, sz, vp]
    lib.vtq_linear_i8_device.restype = i
    lib.vtq_rope_plan.argtypes = [vp, vp, vp]
    lib.vtq_rope_plan.restype = i
    lib.vtq_rope_device.argtypes = [vp, vp, i, vp, sz, sz, vp, sz, sz, vp, sz, sz, sz, vp]
    lib.vtq_rope_device.restype = i
    lib.vtq_kv_append_device.argtypes = [vp, vp, vp, vp, i, sz, vp, sz, sz, vp, sz, sz, sz, vp, sz, sz, vp, sz, sz, vp]
    lib.vtq_kv_append_device.restype = i
    lib.vtq_attention_workspace.argtypes = [vp, vp, i, sz, sz]
    lib.vtq_attention_workspace.restype = sz
    lib.vtq_attention_device.argtypes = [vp, vp, vp, i, sz, sz, vp, sz, sz, vp, sz, sz, vp, ctypes.c_float, vp, sz, vp]
    lib.vtq_attention_device.restype = i
    _lib = lib
    return lib


EXPORTED = (
    "vtq_create", "vtq_destroy", "vtq_last_error", "vtq_version", "vtq_linear",
    "vtq_linear_q4_k_integer", "vtq_linear_q6_k_integer", "vtq_linear_q4_k_fused",
    "vtq_linear_q4_0", "vtq_release_weights", "vtq_linear_device", "vtq_linear_device_noalloc",
    "vtq_quantize_i8_device", "vtq_linear_i8_device", "vtq_rope_plan", "vtq_rope_device", "vtq_kv_append_device",
    "vtq_attention_workspace", "vtq_attention_device",
)


def _fits(lo, hi, **values):
    """Refuses what a C integer would not hold: ctypes cuts it without a word."""
    for name, value in values.items():
        if not lo <= int(value) < hi:
            raise InvalidArgument(f"vtq: {name} does not fit its C type")


def _ints(**values):
    _fits(-(1 << 31), 1 << 31, **values)


class _RopeParams(ctypes.Structure):
    _fields_ = [("layout", ctypes.c_int), ("scaling", ctypes.c_int), ("rot_dim", ctypes.c_int),
                ("original_context", ctypes.c_int), ("theta", ctypes.c_double), ("factor", ctypes.c_double),
                ("low", ctypes.c_double), ("high", ctypes.c_double), ("magnitude", ctypes.c_double),
                ("factors", ctypes.c_void_p)]


class _RopePlan(ctypes.Structure):
    _fields_ = [("layout", ctypes.c_int), ("rot_dim", ctypes.c_int), ("magnitude", ctypes.c_float),
                ("reserved", ctypes.c_int), ("turns", ctypes.c_uint64 * 128)]


class _KvCache(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int), ("page_size", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("n_pages", ctypes.c_size_t), ("k", ctypes.c_void_p),
                ("v", ctypes.c_void_p), ("page_stride", ctypes.c_size_t), ("head_stride", ctypes.c_size_t),
                ("slot_stride", ctypes.c_size_t)]


class _KvBatch(ctypes.Structure):
    _fields_ = [("batch", ctypes.c_int), ("max_pages", ctypes.c_int), ("max_q", ctypes.c_int),
                ("max_len", ctypes.c_int), ("prefix_len", ctypes.c_int), ("q_start", ctypes.c_void_p),
                ("len", ctypes.c_void_p), ("pages", ctypes.c_void_p), ("prefix_pages", ctypes.c_void_p)]


class Rope:
    """A rotary plan (vtq_rope_plan): the rot_dim / 2 frequencies and the magnitude.  Host memory, made
    without a device; any context may use it."""

    def __init__(self, rot_dim, layout=ROPE_HALF, theta=10000.0, scaling=ROPE_SCALE_NONE, factor=1.0,
                 original_context=0, low=0.0, high=0.0, magnitude=0.0, factors=None):
        lib = load_library()
        _ints(layout=layout, scaling=scaling, rot_dim=rot_dim, original_context=original_context)
        f = None if factors is None else np.ascontiguousarray(factors, dtype=np.float32)
        if f is not None and f.size != int(rot_dim) // 2:
            raise InvalidShape("vtq: one rope factor a pair")
        params = _RopeParams(layout, scaling, rot_dim, original_context, theta, factor, low, high, magnitude,
                             None if f is None else f.ctypes.data)
        self.plan = _RopePlan()
        rc = lib.vtq_rope_plan(None, ctypes.byref(params), ctypes.byref(self.plan))
        if rc != OK:
            raise _ERRORS.get(rc, VtqError)("vtq: invalid rope parameters")
        self.ref = ctypes.byref(self.plan)


class KvCache:
    """A paged KV cache on the device (vtq_kv_cache): pages x kv_heads x page_size x head_dim, or the
    given strides in elements.  Holds addresses, not the memory."""

    def __init__(self, ggml_type, k_ptr, v_ptr, n_pages, page_size, kv_heads, head_dim, page_stride=None,
                 head_stride=None, slot_stride=None):
        slot = head_dim if slot_stride is None else slot_stride
        head = page_size * slot if head_stride is None else head_stride
        page = kv_heads * head if page_stride is None else page_stride
        _ints(ggml_type=ggml_type, page_size=page_size, kv_heads=kv_heads, head_dim=head_dim)
        _fits(0, 1 << 64, n_pages=n_pages, page_stride=page, head_stride=head, slot_stride=slot)
        self.desc = _KvCache(int(ggml_type), page_size, kv_heads, head_dim, n_pages, k_ptr, v_ptr, page, head, slot)
        self.ref = ctypes.byref(self.desc)


class KvBatch:
    """A ragged batch over a paged cache (vtq_kv_batch); the pointers are int32 lists on the device."""

    def __init__(self, batch, q_start_ptr, len_ptr, pages_ptr, max_pages, max_q=1, max_len=0, prefix_len=0,
                 prefix_pages=None):
        _ints(batch=batch, max_pages=max_pages, max_q=max_q, max_len=max_len, prefix_len=prefix_len)
        self.desc = _KvBatch(batch, max_pages, max_q, max_len, prefix_len, q_start_ptr, len_ptr, pages_ptr,
                             prefix_pages)
        self.ref = ctypes.byref(self.desc)


class Context:
    """One libvtq context (one HIP device, used by one thread at a time).

    Host-pointer calls cache the weight bytes on the device keyed by the
    array's address and length, as the reference's weights are immutable
    views into a GGUF blob.  Call release_weights() before reusing or freeing
    a weight array whose bytes change.
    """

    def __init__(self, device: int = 0):
        self.lib = load_library()
        h = ctypes.c_void_p()
        rc = self.lib.vtq_create(int(device), ctypes.byref(h))
        if rc != OK:
            raise GpuError(f"vtq_create({device}) failed with status {rc}: no usable HIP device")
        self.handle = h
        self.device = device

    def close(self) -> None:
        if getattr(self, "handle", None):
            self.lib.vtq_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def _check(self, rc: int) -> None:
        if rc == OK:
            return
        msg = self.lib.vtq_last_error(self.handle).decode(errors="replace")
        raise _ERRORS.get(rc, VtqError)(msg)

    # -- host-pointer calls -------------------------------------------------

    @staticmethod
    def _f32(a: np.ndarray, name: str) -> np.ndarray:
        if not isinstance(a, np.ndarray) or a.dtype != np.float32 or not a.flags.c_contiguous:
            raise TypeError(f"{name} must be a C-contiguous float32 numpy array")
        return a

    @staticmethod
    def _u8(a) -> np.ndarray:
        if isinstance(a, (bytes, bytearray)):
            a = np.frombuffer(a, dtype=np.uint8)
        if not isinstance(a, np.ndarray) or a.dtype != np.uint8 or not a.flags.c_contiguous:
            raise TypeError("w must be a C-contiguous uint8 numpy array or bytes")
        return a

    def _host(self, fn, x, w, y_out, batch, in_feat, out_feat):
        x = self._f32(x, "x")
        y_out = self._f32(y_out, "y_out")
        w = self._u8(w)
        if not y_out.flags.writeable:
            raise TypeError("y_out must be writeable")
        rc = fn(self.handle, x.ctypes.data, x.size, w.ctypes.data, w.size, y_out.ctypes.data, y_out.size,
                batch, in_feat, out_feat)
        self._check(rc)

    def linear_q4_k_integer(self, x, w_q4k, y_out, batch, in_feat, out_feat):
        """src/ops/quant.rs:936-980"""
        self._host(self.lib.vtq_linear_q4_k_integer, x, w_q4k, y_out, batch, in_feat, out_feat)

    def linear_q6_k_integer(self, x, w_q6k, y_out, batch, in_feat, out_feat):
        """src/ops/quant.rs:1060-1096"""
        self._host(self.lib.vtq_linear_q6_k_integer, x, w_q6k, y_out, batch, in_feat, out_feat)

    def linear_q4_k_fused(self, x, w_q4k, y_out, batch, in_feat, out_feat):
        """src/ops/quant.rs:1433-1453"""
        self._host(self.lib.vtq_linear_q4_k_fused, x, w_q4k, y_out, batch, in_feat, out_feat)

    def linear_q4_0(self, x, w_q4, y_out, batch, in_feat, out_feat):
        """src/ops/quant.rs:1529-1565 (linear_q4_0_cpu)"""
        self._host(self.lib.vtq_linear_q4_0, x, w_q4, y_out, batch, in_feat, out_feat)

    def linear(self, ggml_type, regime, x, w, y_out, batch, in_feat, out_feat):
        """src/model/forward_quantized.rs:663-785 (linear_dispatch), any batch."""
        x = self._f32(x, "x")
        y_out = self._f32(y_out, "y_out")
        w = self._u8(w)
        rc = self.lib.vtq_linear(self.handle, int(ggml_type), int(regime), x.ctypes.data, x.size, w.ctypes.data,
                                 w.size, y_out.ctypes.data, y_out.size, batch, in_feat, out_feat)
        self._check(rc)

    def linear_dispatch(self, x, w, ggml_type, in_feat, out_feat, regime=REGIME_INTEGER):
        """The reference's linear_dispatch shape: batch 1, returns a new y."""
        y = np.zeros(out_feat, dtype=np.float32)
        self.linear(ggml_type, regime, x, w, y, 1, in_feat, out_feat)
        return y

    def release_weights(self, w=None):
        ptr = None if w is None else self._u8(w).ctypes.data
        self._check(self.lib.vtq_release_weights(self.handle, ptr))

    # -- device-pointer call ------------------------------------------------

    def linear_device(self, ggml_type, regime, x_ptr, w_ptr, w_len, y_ptr, batch, in_feat, out_feat, stream=None):
        """Enqueue on `stream` (int handle or None); pointers are device addresses."""
        rc = self.lib.vtq_linear_device(self.handle, int(ggml_type), int(regime), x_ptr, w_ptr, w_len, y_ptr,
                                        batch, in_feat, out_feat, stream)
        self._check(rc)

    # -- operators of a batched serving step (device pointers) ---------------

    def quantize_i8_device(self, x_type, x_ptr, ld_x, q_ptr, ld_q, scale_ptr, rows, n, stream=None):
        """vtq_quantize_i8_device: rows of x to 8 bits with a scale each."""
        rc = self.lib.vtq_quantize_i8_device(self.handle, x_type, x_ptr, ld_x, q_ptr, ld_q, scale_ptr, rows, n, stream)
        if rc:
            self._check(rc)

    def linear_i8_device(self, xq_ptr, ld_x, x_scale_ptr, wq_ptr, ld_w, w_scale_ptr, bias_ptr, y_type, y_ptr, ld_y,
                         batch, in_feat, out_feat, stream=None):
        """vtq_linear_i8_device: the int8 product with scales per token and channel."""
        rc = self.lib.vtq_linear_i8_device(self.handle, xq_ptr, ld_x, x_scale_ptr, wq_ptr, ld_w, w_scale_ptr, bias_ptr,
                                           y_type, y_ptr, ld_y, batch, in_feat, out_feat, stream)
        if rc:
            self._check(rc)

    def rope_device(self, rope, ggml_type, x_ptr, x_token_stride, x_head_stride, y_ptr, y_token_stride, y_head_stride,
                    pos_ptr, tokens, heads, head_dim, stream=None):
        """vtq_rope_device: x rotated to its positions, into y (or in place)."""
        rc = self.lib.vtq_rope_device(self.handle, rope.ref, ggml_type, x_ptr, x_token_stride, x_head_stride, y_ptr,
                                      y_token_stride, y_head_stride, pos_ptr, tokens, heads, head_dim, stream)
        if rc:
            self._check(rc)

    def kv_append_device(self, cache, batch, rope, ggml_type, tokens, k_ptr, k_token_stride, k_head_stride, v_ptr,
                         v_token_stride, v_head_stride, stream=None, heads=0, q_ptr=None, q_token_stride=0,
                         q_head_stride=0, q_out_ptr=None, q_out_token_stride=0, q_out_head_stride=0):
        """vtq_kv_append_device: rotated keys and plain values to their slots, rotated queries to q_out."""
        rc = self.lib.vtq_kv_append_device(self.handle, cache.ref, batch.ref, None if rope is None else rope.ref,
                                           ggml_type, tokens, k_ptr, k_token_stride, k_head_stride, v_ptr,
                                           v_token_stride, v_head_stride, heads, q_ptr, q_token_stride, q_head_stride,
                                           q_out_ptr, q_out_token_stride, q_out_head_stride, stream)
        if rc:
            self._check(rc)

    def attention_workspace(self, cache, batch, ggml_type, tokens, heads):
        """vtq_attention_workspace: bytes that attention_device needs for these numbers."""
        return self.lib.vtq_attention_workspace(cache.ref, batch.ref, ggml_type, tokens, heads)

    def attention_device(self, cache, batch, ggml_type, tokens, heads, q_ptr, q_token_stride, q_head_stride, y_ptr,
                         y_token_stride, y_head_stride, scale, ws_ptr, ws_bytes, stream=None, lse_ptr=None):
        """vtq_attention_device: attention over the shared prefix and the sequences' own pages."""
        rc = self.lib.vtq_attention_device(self.handle, cache.ref, batch.ref, ggml_type, tokens, heads, q_ptr,
                                           q_token_stride, q_head_stride, y_ptr, y_token_stride, y_head_stride, lse_ptr,
                                           scale, ws_ptr, ws_bytes, stream)
        if rc:
            self._check(rc)


def row_bytes(ggml_type: int, in_feat: int) -> int:
    if ggml_type == F32:
        return 4 * in_feat
    numel, nbytes = BLOCK[ggml_type]
    return (in_feat // numel) * nbytes
