"""What the serving operators refuse, asked without a GPU (libvtq_probe.so holds the same checks)."""
import ctypes

import numpy as np
import pytest

import vtq
from vtq import probe

A = 1 << 20  # an aligned address; nothing is read
OK, ARG, SHAPE, NIMP = vtq.OK, vtq.E_INVALID_ARGUMENT, vtq.E_INVALID_SHAPE, vtq.E_NOT_IMPLEMENTED


def _with(base, **changes):
    d = dict(base)
    for k in changes:
        assert k in d, k
    d.update(changes)
    return list(d.values())


QUANT = dict(type=vtq.F32, x=A, ld_x=100, q=A, ld_q=112, scale=A, rows=3, n=100)


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(type=vtq.Q8_0), NIMP), (dict(type=7), NIMP), (dict(n=131072, ld_x=131072, ld_q=131072), NIMP),
    (dict(ld_q=100), SHAPE), (dict(ld_q=96), SHAPE), (dict(ld_x=99), SHAPE), (dict(ld_x=1, rows=1), OK),
    (dict(rows=0, x=None, q=None, scale=None), OK), (dict(x=None), ARG), (dict(q=None), ARG), (dict(scale=None), ARG),
    (dict(q=A + 8), ARG), (dict(x=A + 2), ARG), (dict(type=vtq.BF16, x=A + 2), OK), (dict(rows=1 << 40), NIMP)])
def test_quantize(change, code):
    rc, text = probe.refusal("quantize_i8", *_with(QUANT, **change))
    assert rc == code and (text != "") == (code != OK)


LINEAR = dict(xq=A, ld_x=112, xs=A, wq=A, ld_w=112, ws=A, bias=None, type=vtq.BF16, y=A, ld_y=64, batch=3, in_feat=100,
              out_feat=64)


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(bias=A), OK), (dict(bias=A + 1), ARG), (dict(type=vtq.Q4_K), NIMP), (dict(in_feat=131072), NIMP),
    (dict(ld_x=100), SHAPE), (dict(ld_w=96), SHAPE), (dict(ld_y=63), SHAPE), (dict(ld_y=1, batch=1), OK),
    (dict(xq=None), ARG), (dict(wq=None), ARG), (dict(xs=None), ARG), (dict(ws=None), ARG), (dict(y=None), ARG),
    (dict(in_feat=0, xq=None, wq=None, xs=None, ws=None), OK), (dict(batch=0, y=None), OK), (dict(out_feat=0, y=None), OK),
    (dict(xq=A + 4), ARG), (dict(wq=A + 8), ARG), (dict(y=A + 1), ARG), (dict(y=A + 2), OK),
    (dict(ld_w=1 << 22), NIMP), (dict(batch=1 << 31), NIMP)])
def test_linear(change, code):
    rc, text = probe.refusal("linear_i8", *_with(LINEAR, **change))
    assert rc == code and (text != "") == (code != OK)


def test_rope_plans():
    for args in (dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=258)):
        with pytest.raises(vtq.InvalidShape):
            vtq.Rope(**args)
    nan, inf = float("nan"), float("inf")
    for args in (dict(layout=2), dict(scaling=4), dict(scaling=-1), dict(theta=1.0), dict(theta=nan), dict(theta=inf),
                 dict(magnitude=-1.0), dict(magnitude=nan),
                 dict(magnitude=1e39), dict(scaling=vtq.ROPE_SCALE_LINEAR, factor=0.5),
                 dict(scaling=vtq.ROPE_SCALE_LINEAR, factor=nan),
                 dict(scaling=vtq.ROPE_SCALE_YARN, factor=2.0, original_context=0),
                 dict(scaling=vtq.ROPE_SCALE_BANDS, factor=2.0, original_context=4096, low=4.0, high=4.0),
                 dict(scaling=vtq.ROPE_SCALE_BANDS, factor=2.0, original_context=4096, low=-1.0),
                 dict(factors=[0.0] * 32), dict(factors=[nan] * 32)):
        with pytest.raises(vtq.InvalidArgument):
            vtq.Rope(64, **args)
    with pytest.raises(vtq.InvalidShape):
        vtq.Rope(64, factors=[1.0] * 31)


def test_rope_frequencies_are_whole_fractions_of_a_turn():
    from serving import frequencies

    for args, plain in ((dict(theta=1e6), dict(theta=1e6)),
                        (dict(scaling=vtq.ROPE_SCALE_LINEAR, factor=4.0),) * 2,
                        (dict(theta=5e5, scaling=vtq.ROPE_SCALE_BANDS, factor=8.0, original_context=8192),
                         dict(theta=5e5, scaling=vtq.ROPE_SCALE_BANDS, factor=8.0, original=8192)),
                        (dict(theta=1e6, scaling=vtq.ROPE_SCALE_YARN, factor=16.0, original_context=8192),
                         dict(theta=1e6, scaling=vtq.ROPE_SCALE_YARN, factor=16.0, original=8192))):
        plan = vtq.Rope(128, **args).plan
        f, m = frequencies(128, **plain)
        got = np.array([plan.turns[i] for i in range(64)], dtype=np.float64) / 2.0 ** 64 * 2 * np.pi
        # a fraction is cut at 2^-64 turn, 2 pi 2^-64 = 3.41e-19 radian; exp and log are off by a few 2^-53 of
        # an exponent up to 14
        assert np.allclose(got, f.numpy(), rtol=1e-13, atol=3.5e-19) and abs(plan.magnitude - m) < 1e-6
    # a factor that makes a pair turn more than once a position: whole turns do not count
    plan = vtq.Rope(2, factors=[1.0 / (2 * np.pi * 3.25)]).plan
    assert abs(plan.turns[0] / 2.0 ** 64 - 0.25) < 1e-6


def _rope_args(**change):
    base = dict(rope=vtq.Rope(64).ref, type=vtq.F32, x=A, xt=640, xh=64, y=A + (1 << 20), yt=640, yh=64, pos=A, tokens=5,
                heads=10, head_dim=64)
    return _with(base, **change)


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(rope=None), ARG), (dict(type=2), NIMP), (dict(head_dim=62), SHAPE), (dict(head_dim=8200), NIMP),
    (dict(x=None), ARG), (dict(y=None), ARG), (dict(pos=None), ARG), (dict(pos=A + 2), ARG), (dict(x=A + 2), ARG),
    (dict(tokens=0, x=None), OK), (dict(heads=0, x=None), OK), (dict(xh=63), SHAPE), (dict(yt=63), SHAPE),
    (dict(y=A), OK), (dict(y=A, yt=700), SHAPE), (dict(tokens=(1 << 23) + 1), NIMP), (dict(heads=65536), NIMP)])
def test_rope_calls(change, code):
    rc, text = probe.refusal("rope_call", *_rope_args(**change))
    assert rc == code and (text != "") == (code != OK)


def _cache(**change):
    base = dict(ggml_type=vtq.BF16, k_ptr=A, v_ptr=A, n_pages=10, page_size=16, kv_heads=2, head_dim=64,
                page_stride=None, head_stride=None, slot_stride=None)
    base.update(change)
    return vtq.KvCache(**base)


def _batch(**change):
    base = dict(batch=2, q_start_ptr=A, len_ptr=A, pages_ptr=A, max_pages=4, max_q=1, max_len=0, prefix_len=5,
                prefix_pages=A)
    base.update(change)
    return vtq.KvBatch(**base)


BAD_CACHES = [(dict(ggml_type=vtq.Q8_0), NIMP), (dict(page_size=4), SHAPE), (dict(page_size=24), SHAPE),
              (dict(page_size=8192), SHAPE), (dict(page_size=0), SHAPE), (dict(head_dim=60), SHAPE),
              (dict(head_dim=264), SHAPE), (dict(head_dim=0), SHAPE), (dict(kv_heads=0), SHAPE),
              (dict(n_pages=1 << 31), NIMP), (dict(slot_stride=68), SHAPE), (dict(slot_stride=56), SHAPE),
              (dict(head_stride=56), SHAPE), (dict(head_stride=4), SHAPE), (dict(page_stride=100), SHAPE),
              (dict(slot_stride=1 << 24), NIMP), (dict(page_size=4096, slot_stride=1 << 17), NIMP),
              (dict(n_pages=2 ** 31 - 1, page_stride=1 << 16), NIMP), (dict(head_stride=1 << 38, page_stride=1024), NIMP),
              (dict(k_ptr=None), ARG), (dict(v_ptr=None), ARG),
              (dict(k_ptr=A + 8), ARG), (dict(v_ptr=A + 2), ARG)]
BAD_BATCHES = [(dict(batch=-1), ARG), (dict(max_pages=-1), ARG), (dict(prefix_len=-1), ARG), (dict(max_q=-1), ARG),
               (dict(max_len=-1), ARG), (dict(batch=(1 << 20) + 1), NIMP), (dict(max_pages=1 << 28), NIMP),
               (dict(prefix_len=1 << 30), NIMP), (dict(q_start_ptr=None), ARG), (dict(len_ptr=None), ARG),
               (dict(pages_ptr=None), ARG), (dict(q_start_ptr=A + 2), ARG), (dict(len_ptr=A + 1), ARG),
               (dict(pages_ptr=A + 2), ARG)]


def _append_args(cache=None, batch=None, **change):
    base = dict(cache=(cache or _cache()).ref, batch=(batch or _batch()).ref, rope=vtq.Rope(64).ref, type=vtq.BF16,
                tokens=3, k=A, kt=128, kh=64, v=A, vt=128, vh=64, heads=4, q=A, qt=256, qh=64, out=A + 65536, ot=256,
                oh=64)
    return _with(base, **change)


def _attention_args(cache=None, batch=None, **change):
    base = dict(cache=(cache or _cache()).ref, batch=(batch or _batch()).ref, type=vtq.BF16, tokens=3, heads=4, q=A,
                qt=256, qh=64, y=A, yt=256, yh=64, lse=None, scale=0.125)
    return _with(base, **change)


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_caches(change, code):
    for operator, args in (("append", _append_args), ("attention", _attention_args)):
        rc, text = probe.refusal(operator, *args(cache=_cache(**change)))
        assert rc == code and text, (operator, text)
    lib = vtq.load_library()
    assert lib.vtq_attention_workspace(_cache(**change).ref, _batch().ref, vtq.BF16, 3, 4) == 0


@pytest.mark.parametrize("change,code", BAD_BATCHES)
def test_batches(change, code):
    for operator, args in (("append", _append_args), ("attention", _attention_args)):
        rc, text = probe.refusal(operator, *args(batch=_batch(**change)))
        assert rc == code and text, (operator, text)


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(cache=None), ARG), (dict(batch=None), ARG), (dict(rope=None), OK), (dict(type=vtq.F32), OK),
    (dict(type=vtq.F16), NIMP), (dict(type=2), NIMP), (dict(k=None), ARG), (dict(v=None), ARG), (dict(q=None), OK),
    (dict(heads=0), OK), (dict(out=None), ARG), (dict(out=A), OK), (dict(out=A, ot=300), SHAPE), (dict(kh=56), SHAPE),
    (dict(vt=40), SHAPE), (dict(qh=8), SHAPE), (dict(tokens=0, k=None), OK), (dict(k=A + 1), ARG),
    (dict(tokens=(1 << 23) + 1), NIMP)])
def test_append(change, code):
    args = _append_args(**{k: v for k, v in change.items() if k not in ("cache", "batch")})
    if "cache" in change:
        args[0] = None
    if "batch" in change:
        args[1] = None
    rc, text = probe.refusal("append", *args)
    assert rc == code and (text != "") == (code != OK)
    assert probe.refusal("append", *_append_args(rope=vtq.Rope(128).ref))[0] == SHAPE  # rot_dim beyond head_dim
    # only attention reads the prefix
    assert probe.refusal("append", *_append_args(batch=_batch(prefix_pages=None)))[0] == OK


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(type=vtq.F32, qt=256), OK), (dict(type=vtq.F16), NIMP), (dict(heads=3), SHAPE), (dict(q=None), ARG),
    (dict(y=None), ARG), (dict(q=A + 8), ARG), (dict(y=A + 2), ARG), (dict(qt=260), ARG), (dict(yh=68), ARG),
    (dict(qh=56), SHAPE), (dict(lse=A), OK), (dict(lse=A + 2), ARG), (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG),
    (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG), (dict(scale=2e30), ARG), (dict(tokens=0, q=None), OK),
    (dict(heads=0, q=None), OK), (dict(heads=65536), NIMP), (dict(y=A, yt=512), SHAPE),
    (dict(y=A + 65536, yt=512), OK)])
def test_attention(change, code):
    rc, text = probe.refusal("attention", *_attention_args(**change))
    assert rc == code and (text != "") == (code != OK)
    for address in (None, A + 2):
        assert probe.refusal("attention", *_attention_args(batch=_batch(prefix_pages=address)))[0] == ARG


def test_heads_before_pages_are_taken():
    cache = _cache(n_pages=1 << 16, page_stride=16 * 64, head_stride=(1 << 16) * 16 * 64)
    for operator, args in (("append", _append_args), ("attention", _attention_args)):
        assert probe.refusal(operator, *args(cache=cache)) == (OK, "")


def test_null_contexts_are_refused():
    lib = vtq.load_library()
    assert lib.vtq_quantize_i8_device(None, *_with(QUANT), None) == ARG
    assert lib.vtq_linear_i8_device(None, *_with(LINEAR), None) == ARG
    assert lib.vtq_rope_device(None, *_rope_args(), None) == ARG
    assert lib.vtq_kv_append_device(None, *_append_args(), None) == ARG
    assert lib.vtq_attention_device(None, *_attention_args(), None, 0, None) == ARG
    assert lib.vtq_rope_plan(None, None, None) == ARG


def test_places_without_a_slot():
    pages = (ctypes.c_int32 * 4)(7, -1, 10, 2 ** 31 - 1)
    cache = _cache()
    at = lambda place: probe.lib().vtqp_slot_of(cache.ref, pages, 4, place)  # noqa: E731
    assert at(0) == 7 * 2 * 16 * 64 and at(15) == 7 * 2 * 16 * 64 + 15 * 64
    for place in (-1, -2 ** 40, 16, 31, 32, 48, 63, 64, 2 ** 40):  # before, pages -1, 10 (of 10), 2^31 - 1, past
        assert at(place) == -1, place
    far = _cache(n_pages=2 ** 31 - 1, page_stride=1 << 15)
    pages[0] = 2 ** 31 - 2
    assert probe.lib().vtqp_slot_of(far.ref, pages, 4, 3) == (2 ** 31 - 2) * (1 << 15) + 3 * 64
