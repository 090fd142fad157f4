"""What the Python binding of the serving operators refuses itself: numbers that a C int does not hold, which ctypes
would cut to 32 bits without a word."""
import pytest

import vtq

A = 1 << 20  # an aligned address; nothing is read
CACHE = dict(ggml_type=vtq.BF16, k_ptr=A, v_ptr=A, n_pages=10, page_size=16, kv_heads=2, head_dim=64)
BATCH = dict(batch=2, q_start_ptr=A, len_ptr=A, pages_ptr=A, max_pages=4, max_q=1, max_len=0, prefix_len=5,
             prefix_pages=A)
ROPE = dict(rot_dim=64, layout=vtq.ROPE_HALF, scaling=vtq.ROPE_SCALE_NONE, original_context=4096)


@pytest.mark.parametrize("make,base,names", [
    (vtq.KvCache, CACHE, ("ggml_type", "page_size", "kv_heads", "head_dim")),
    (vtq.KvBatch, BATCH, ("batch", "max_pages", "max_q", "max_len", "prefix_len")),
    (vtq.Rope, ROPE, ("rot_dim", "layout", "scaling", "original_context"))])
@pytest.mark.parametrize("past", [1 << 32, 1 << 31, -(1 << 32), -(1 << 31) - 1])
def test_numbers_past_a_c_int_are_refused(make, base, names, past):
    make(**base)
    for name in names:
        value = past + base[name] if abs(past) == 1 << 32 else past
        with pytest.raises(vtq.InvalidArgument):
            make(**{**base, name: value})


def test_strides_and_counts_past_a_size_t_are_refused():
    for name in ("n_pages", "page_stride", "head_stride", "slot_stride"):
        for value in (1 << 64, -1):
            with pytest.raises(vtq.InvalidArgument):
                vtq.KvCache(**{**CACHE, name: value})
