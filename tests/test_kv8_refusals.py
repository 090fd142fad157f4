"""What the operators over 8-bit caches, the selection of beams and the pages' operators refuse, asked without a GPU
(libvtq_probe.so holds the same checks), and what their Python binding refuses itself."""
import pytest

import vtq
from test_serve_refusals import BAD_BATCHES, A, _batch, _with
from vtq import probe

OK, ARG, SHAPE, NIMP = vtq.OK, vtq.E_INVALID_ARGUMENT, vtq.E_INVALID_SHAPE, vtq.E_NOT_IMPLEMENTED


def _cache8(type_=None, **change):
    base = dict(k_ptr=A, v_ptr=A, k_scale_ptr=A, v_scale_ptr=A + 1, n_pages=10, page_size=32, kv_heads=2, head_dim=64,
                block=16, page_stride=None, head_stride=None, slot_stride=None, scale_page_stride=None,
                scale_head_stride=None)
    base.update(change)
    c = vtq.Kv8Cache(**base)
    if type_ is not None:
        c.desc.cache.type = type_
    return c


def _append_args(cache=None, batch=None, **change):
    base = dict(cache=(cache or _cache8()).ref, batch=(batch or _batch()).ref, rope=vtq.Rope(64).ref, type=vtq.BF16,
                tokens=3, k=A, kt=128, kh=64, v=A, vt=128, vh=64, heads=4, q=A, qt=256, qh=64, out=A + 65536, ot=256,
                oh=64)
    return _with(base, **change)


def _attention_args(cache=None, batch=None, **change):
    base = dict(cache=(cache or _cache8()).ref, batch=(batch or _batch()).ref, type=vtq.BF16, tokens=3, heads=4, q=A,
                qt=256, qh=64, y=A, yt=256, yh=64, lse=None, scale=0.125)
    return _with(base, **change)


BAD_CACHES = [
    (dict(type_=vtq.BF16), NIMP), (dict(type_=24), NIMP), (dict(page_size=8, block=8), SHAPE), (dict(page_size=48), SHAPE),
    (dict(page_size=8192), SHAPE), (dict(head_dim=72), SHAPE), (dict(head_dim=8), SHAPE), (dict(head_dim=272), SHAPE),
    (dict(head_dim=0), SHAPE), (dict(kv_heads=0), SHAPE), (dict(block=8), SHAPE), (dict(block=64), SHAPE),
    (dict(block=24), SHAPE), (dict(block=-16), SHAPE), (dict(slot_stride=72), SHAPE), (dict(slot_stride=48), SHAPE),
    (dict(head_stride=2056), SHAPE), (dict(page_stride=4104), SHAPE), (dict(scale_head_stride=1), SHAPE),
    (dict(scale_page_stride=1, scale_head_stride=2), SHAPE), (dict(n_pages=1 << 31), NIMP),
    (dict(slot_stride=1 << 24), NIMP), (dict(scale_page_stride=1 << 38), NIMP), (dict(scale_head_stride=1 << 38), NIMP),
    (dict(n_pages=2 ** 31 - 1, scale_page_stride=1 << 17), NIMP), (dict(k_ptr=None), ARG), (dict(v_ptr=None), ARG),
    (dict(k_ptr=A + 8), ARG), (dict(k_scale_ptr=None), ARG), (dict(v_scale_ptr=None), ARG)]


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_caches(change, code):
    for operator, args in (("kv8_append", _append_args), ("kv8_attention", _attention_args)):
        rc, text = probe.refusal(operator, *args(cache=_cache8(**change)))
        assert rc == code and text, (operator, text)
    rc, text = probe.refusal("kv8_pages_copy", _cache8(**change).ref, 1, 0, 0, A, 3, None)
    assert rc == code and text
    assert vtq.load_library().vtq_kv8_attention_workspace(_cache8(**change).ref, _batch().ref, vtq.BF16, 3, 4) == 0


def test_the_wider_operators_refuse_an_8_bit_cache():
    cache = vtq.KvCache(vtq.E4M3, A, A, 10, 16, 2, 64)
    assert probe.refusal("append", cache.ref, _batch().ref, None, vtq.F32, 3, A, 128, 64, A, 128, 64, 0, None, 0, 0, None,
                         0, 0)[0] == NIMP
    assert probe.refusal("attention", cache.ref, *_attention_args()[1:])[0] == NIMP
    assert probe.refusal("pages_copy", cache.ref, 1, 0, A, 3, None)[0] == NIMP


@pytest.mark.parametrize("change,code", BAD_BATCHES)
def test_batches(change, code):
    for operator, args in (("kv8_append", _append_args), ("kv8_attention", _attention_args)):
        rc, text = probe.refusal(operator, *args(batch=_batch(**change)))
        assert rc == code and text, (operator, text)


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(rope=None), OK), (dict(type=vtq.F32), OK), (dict(type=vtq.F16), OK), (dict(type=vtq.E4M3), NIMP),
    (dict(type=2), NIMP), (dict(k=None), ARG), (dict(v=None), ARG), (dict(q=None), OK), (dict(heads=0), OK),
    (dict(out=None), ARG), (dict(out=A), OK), (dict(out=A, ot=300), SHAPE), (dict(kh=56), SHAPE), (dict(vt=40), SHAPE),
    (dict(qh=8), SHAPE), (dict(tokens=0, k=None), OK), (dict(k=A + 1), ARG), (dict(tokens=(1 << 23) + 1), NIMP)])
def test_append(change, code):
    rc, text = probe.refusal("kv8_append", *_append_args(**change))
    assert rc == code and (text != "") == (code != OK)
    assert probe.refusal("kv8_append", *_append_args(rope=vtq.Rope(128).ref))[0] == SHAPE  # rot_dim beyond head_dim
    assert probe.refusal("kv8_append", *_append_args(cache=_cache8(kv_heads=1 << 10), tokens=(1 << 16) + 1, kt=1 << 16,
                                                     vt=1 << 16))[0] == NIMP  # more than 2^26 keys
    assert probe.refusal("kv8_append", None, *_append_args()[1:])[0] == ARG
    assert probe.refusal("kv8_append", _append_args()[0], None, *_append_args()[2:])[0] == ARG


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(type=vtq.F32), OK), (dict(type=vtq.F16), OK), (dict(type=vtq.E4M3), NIMP), (dict(heads=3), SHAPE),
    (dict(q=None), ARG), (dict(y=None), ARG), (dict(q=A + 8), ARG), (dict(y=A + 2), ARG), (dict(qt=260), ARG),
    (dict(yh=68), ARG), (dict(qh=56), SHAPE), (dict(lse=A), OK), (dict(lse=A + 2), ARG), (dict(scale=0.0), ARG),
    (dict(scale=float("nan")), ARG), (dict(scale=2e30), ARG), (dict(tokens=0, q=None), OK), (dict(heads=0, q=None), OK),
    (dict(heads=65536), NIMP), (dict(y=A, yt=512), SHAPE), (dict(y=A + 65536, yt=512), OK)])
def test_attention(change, code):
    rc, text = probe.refusal("kv8_attention", *_attention_args(**change))
    assert rc == code and (text != "") == (code != OK)
    for address in (None, A + 2):
        assert probe.refusal("kv8_attention", *_attention_args(batch=_batch(prefix_pages=address)))[0] == ARG


BEAM = dict(type=vtq.F32, logits=A, ld=1000, groups=2, beams=4, vocab=1000, score=A, done=None, end=-1, n_out=8,
            out_score=A + 64, token=A, parent=A, out_done=None)


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(type=vtq.BF16), OK), (dict(type=vtq.E4M3), NIMP), (dict(type=vtq.Q8_0), NIMP), (dict(logits=None), ARG),
    (dict(logits=A + 2), ARG), (dict(type=vtq.F16, logits=A + 2), OK), (dict(ld=999), SHAPE),
    (dict(ld=0, groups=1, beams=1), OK), (dict(ld=1 << 38), NIMP), (dict(groups=0, logits=None), OK), (dict(beams=0), SHAPE),
    (dict(vocab=0), SHAPE), (dict(n_out=0), SHAPE), (dict(beams=65), NIMP), (dict(n_out=65), NIMP),
    (dict(vocab=(1 << 20) + 1, ld=1 << 21), NIMP), (dict(groups=(1 << 18) + 1), NIMP), (dict(groups=1 << 62), NIMP),
    (dict(end=1000), ARG), (dict(end=999), OK), (dict(end=-7), OK), (dict(score=None), ARG), (dict(out_score=None), ARG),
    (dict(token=None), ARG), (dict(parent=None), ARG), (dict(score=A + 1), ARG), (dict(token=A + 2), ARG),
    (dict(done=A + 1, out_done=A + 3), OK), (dict(done=A, out_done=A), SHAPE), (dict(done=A, out_done=A, n_out=4), OK),
    (dict(out_score=A), SHAPE), (dict(out_score=A, n_out=4), OK)])
def test_beam_select(change, code):
    rc, text = probe.refusal("beam_select", *_with(BEAM, **change))
    assert rc == code and (text != "") == (code != OK)


REORDER = dict(n_pages=10, page=16, max_pages=4, refs=A, batch=3, pages=A, len=A, batch_out=5, parent=A, grow=None,
               new_refs=A + 64, new_pages=A + 64, new_len=A + 64, copies=A, info=A)


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(grow=A), OK), (dict(grow=A + 1), ARG), (dict(page=12), SHAPE), (dict(page=0), SHAPE),
    (dict(page=-16), SHAPE), (dict(page=8192), SHAPE), (dict(n_pages=(1 << 24) + 1), NIMP), (dict(n_pages=0, refs=None, new_refs=None), OK),
    (dict(refs=None), ARG), (dict(new_refs=None), ARG), (dict(new_refs=A), ARG), (dict(refs=A + 2), ARG),
    (dict(batch=(1 << 16) + 1), NIMP), (dict(batch_out=(1 << 16) + 1), NIMP), (dict(max_pages=1 << 27), NIMP),
    (dict(max_pages=1 << 62), NIMP), (dict(pages=None), ARG), (dict(len=None), ARG), (dict(batch=0, pages=None, len=None), OK),
    (dict(max_pages=0, pages=None, new_pages=None), OK), (dict(parent=None), ARG), (dict(new_pages=None), ARG),
    (dict(new_len=None), ARG), (dict(copies=None), ARG), (dict(info=None), ARG), (dict(info=A + 2), ARG),
    (dict(batch_out=0, parent=None, new_pages=None, new_len=None, copies=None), OK), (dict(new_pages=A), ARG),
    (dict(new_len=A), ARG), (dict(copies=A + 1), ARG)])
def test_pages_reorder(change, code):
    rc, text = probe.refusal("pages_reorder", *_with(REORDER, **change))
    assert rc == code and (text != "") == (code != OK)


COMPACT = dict(n_pages=10, page=16, refs=A, n_entries=5, pages=A, n_prefix=0, prefix=None, new_refs=A + 64, new_pages=A,
               new_prefix=None, copies=A, info=A)


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(n_prefix=2), ARG), (dict(n_prefix=2, prefix=A, new_prefix=A), OK), (dict(n_entries=0, pages=None,
                                                                                           new_pages=None), OK),
    (dict(pages=None), ARG), (dict(new_pages=None), ARG), (dict(copies=None), ARG), (dict(n_pages=1, copies=None), OK),
    (dict(new_refs=A), ARG), (dict(page=20), SHAPE), (dict(n_entries=1 << 31), NIMP), (dict(n_prefix=1 << 31), NIMP),
    (dict(pages=A + 2), ARG), (dict(info=None), ARG), (dict(refs=None), ARG)])
def test_pages_compact(change, code):
    rc, text = probe.refusal("pages_compact", *_with(COMPACT, **change))
    assert rc == code and (text != "") == (code != OK)


COPY = dict(layers=3, layer_stride=1 << 20, copies=A, max_copies=7, count=None)


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(count=A), OK), (dict(count=A + 1), ARG), (dict(copies=None), ARG), (dict(copies=A + 2), ARG),
    (dict(layers=0, copies=None), OK), (dict(max_copies=0, copies=None), OK), (dict(layers=65536), NIMP),
    (dict(max_copies=1 << 31), NIMP), (dict(layer_stride=0), SHAPE), (dict(layer_stride=0, layers=1), OK),
    (dict(layer_stride=(1 << 20) + 4), SHAPE), (dict(layer_stride=1 << 40), NIMP)])
def test_pages_copy(change, code):
    plain, eight = vtq.KvCache(vtq.F16, A, A, 10, 16, 2, 64), _cache8()
    rc, text = probe.refusal("pages_copy", plain.ref, *_with(COPY, **change))
    assert rc == code and (text != "") == (code != OK)
    args = _with(COPY, **change)
    args.insert(2, 1 << 10)
    rc, text = probe.refusal("kv8_pages_copy", eight.ref, *args)
    assert rc == code and (text != "") == (code != OK)
    assert probe.refusal("pages_copy", None, *_with(COPY))[0] == ARG
    assert probe.refusal("kv8_pages_copy", eight.ref, 3, 1 << 20, 0, A, 7, None)[0] == SHAPE
    assert probe.refusal("kv8_pages_copy", eight.ref, 3, 1 << 20, 1 << 41, A, 7, None)[0] == NIMP
    assert probe.refusal("kv8_pages_copy", eight.ref, 3, (1 << 20) + 8, 64, A, 7, None)[0] == SHAPE
    many = vtq.KvCache(vtq.F16, A, A, 10, 4096, 65535, 64, head_stride=64)
    assert probe.refusal("pages_copy", many.ref, 3, 1 << 20, A, 7, None)[0] == NIMP


def test_workspaces_of_refused_sizes_are_none():
    lib = vtq.load_library()
    assert lib.vtq_beam_select_workspace(2, 4, 1000, 8) > 0
    for sizes in ((0, 4, 1000, 8), (2, 0, 1000, 8), (2, 65, 1000, 8), (2, 4, 1 << 21, 8), (2, 4, 1000, 65),
                  (1 << 20, 2, 10, 1), (1 << 62, 4, 10, 1)):
        assert lib.vtq_beam_select_workspace(*sizes) == 0
    assert lib.vtq_pages_reorder_workspace(10, 3, 5) > 0 and lib.vtq_pages_compact_workspace(10) > 0
    assert lib.vtq_pages_reorder_workspace((1 << 24) + 1, 3, 5) == lib.vtq_pages_reorder_workspace(10, 3, 1 << 17) == 0
    assert lib.vtq_pages_compact_workspace((1 << 24) + 1) == 0
    assert lib.vtq_kv8_attention_workspace(None, None, vtq.BF16, 3, 4) == 0


def test_null_contexts_are_refused():
    lib = vtq.load_library()
    assert lib.vtq_kv8_append_device(None, *_append_args(), None) == ARG
    assert lib.vtq_kv8_attention_device(None, *_attention_args(), None, 0, None) == ARG
    assert lib.vtq_beam_select_device(None, *_with(BEAM), None, 0, None) == ARG
    assert lib.vtq_pages_reorder_device(None, *_with(REORDER), None, 0, None) == ARG
    assert lib.vtq_pages_compact_device(None, *_with(COMPACT), None, 0, None) == ARG
    assert lib.vtq_pages_copy_device(None, None, *_with(COPY), None) == ARG
    assert lib.vtq_kv8_pages_copy_device(None, None, 1, 0, 0, A, 1, None, None) == ARG


@pytest.mark.parametrize("past", [1 << 32, 1 << 31, -(1 << 32), -(1 << 31) - 1])
def test_the_binding_refuses_numbers_past_a_c_int(past):
    for name, value in (("page_size", 32), ("kv_heads", 2), ("head_dim", 64), ("block", 16)):
        with pytest.raises(vtq.InvalidArgument):
            _cache8(**{name: past + value if abs(past) == 1 << 32 else past})
    for name in ("scale_page_stride", "scale_head_stride", "page_stride"):
        with pytest.raises(vtq.InvalidArgument):
            _cache8(**{name: 1 << 64})


def test_the_structs_are_those_of_the_header():
    import ctypes

    assert ctypes.sizeof(vtq._KvCache) == 64 and ctypes.sizeof(vtq._Kv8Cache) == 64 + 8 + 32
