"""Argument checks of the 4-bit cache's and the 4-bit weights' C entry points: refused before any device work."""

import ctypes

import pytest

from maxsim_b200 import _lib
from maxsim_b200._lib import check, lib

_PTR = 1 << 20  # never dereferenced: every call here is refused or has nothing to do


def _cache(**kw):
    c = dict(k_codes=_PTR, k_scales=_PTR, v_codes=_PTR, v_scales=_PTR, num_pages=4, page_size=16, kv_heads=2,
             head_dim=128, device=0)
    c.update(kw)
    return _lib.Kv4Cache(**c)


def _args(**kw):
    a = dict(query=_PTR, query_row_stride=512, query_head_stride=128, rows=2, page_table=_PTR, page_table_stride=3,
             lengths=_PTR, query_offsets=None, out=_PTR, lse=None, workspace=None, workspace_bytes=0, batch=2,
             max_pages=3, max_query_rows=1, heads=4, type=_lib.TYPE_F16, causal=1, window=0, scale=0.1)
    a.update(kw)
    return _lib.Kv4AttendArgs(**a)


def _append(cache, keys=_PTR, values=_PTR, type=_lib.TYPE_F32, tokens=1, slots=_PTR):
    return lib.msb_kv4_append_device(cache if cache is None else ctypes.byref(cache), keys, values, type, tokens, 256,
                                     128, 256, 128, slots, None)


@pytest.mark.parametrize("kw,text", [(dict(k_codes=None), "NULL"), (dict(v_scales=None), "NULL"),
                                     (dict(num_pages=0), "positive"), (dict(kv_heads=0), "positive"),
                                     (dict(num_pages=1 << 31), "num_pages"), (dict(kv_heads=70000), "kv_heads"),
                                     (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"),
                                     (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"),
                                     (dict(k_codes=_PTR + 8), "aligned")])
def test_cache_is_checked_by_every_entry_point(kw, text):
    c = _cache(**kw)
    for status in (_append(c), lib.msb_kv4_read_device(ctypes.byref(c), _PTR, 1, _lib.TYPE_F32, _PTR, _PTR, None),
                   lib.msb_kv4_attend_device(ctypes.byref(c), ctypes.byref(_args()), None)):
        with pytest.raises(ValueError, match=text):
            check(status)


def test_append_and_read_arguments():
    for kw, text in ((dict(keys=None), "NULL"), (dict(slots=None), "NULL"), (dict(type=7), "type must be"),
                     (dict(tokens=-1), "tokens"), (dict(tokens=1 << 31), "tokens")):
        with pytest.raises(ValueError, match=text):
            check(_append(_cache(), **kw))
    with pytest.raises(ValueError, match="cache is NULL"):
        check(_append(None))
    check(_append(_cache(), keys=None, values=None, slots=None, tokens=0))
    check(lib.msb_kv4_read_device(ctypes.byref(_cache()), None, 0, _lib.TYPE_BF16, None, None, None))
    with pytest.raises(ValueError, match="NULL"):
        check(lib.msb_kv4_read_device(ctypes.byref(_cache()), _PTR, 1, _lib.TYPE_BF16, None, _PTR, None))


@pytest.mark.parametrize("kw,text", [(dict(rows=-1), "negative"), (dict(batch=-2), "negative"),
                                     (dict(heads=3), "multiple"), (dict(heads=0), "multiple"),
                                     (dict(rows=3), "rows must equal batch"), (dict(type=_lib.TYPE_F32), "fp16 or bf16"),
                                     (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
                                     (dict(window=-1), "window"), (dict(window=4, causal=0), "window needs causal"),
                                     (dict(max_pages=1 << 28), "max_pages"), (dict(rows=1 << 30, batch=1 << 30), "rows \\* heads"), (dict(query=None), "NULL"),
                                     (dict(lengths=None), "NULL"), (dict(out=None), "NULL"),
                                     (dict(page_table=None), "NULL")])
def test_attend_arguments(kw, text):
    with pytest.raises(ValueError, match=text):
        check(lib.msb_kv4_attend_device(ctypes.byref(_cache()), ctypes.byref(_args(**kw)), None))


def test_tokens_of_a_table_leave_room_past_the_end():
    """Kernels ask for pages some tiles past a sequence's end: positions must not pass 2^31 there."""
    for size in (16, 1024):
        c, a = _cache(page_size=size), _args(max_pages=((1 << 31) - 65536) // size + 1)
        with pytest.raises(ValueError, match="max_pages"):
            check(lib.msb_kv4_attend_device(ctypes.byref(c), ctypes.byref(a), None))


def test_attend_with_nothing_to_do():
    check(lib.msb_kv4_attend_device(ctypes.byref(_cache()), ctypes.byref(_args(rows=0, batch=0, query=None, out=None)), None))


def test_weights():
    a, b = ctypes.c_int64(), ctypes.c_int64()
    check(lib.msb_w4_packed_bytes(17, 136, 64, ctypes.byref(a), ctypes.byref(b)))
    assert (a.value, b.value) == (2 * 3 * 512, 2 * 3 * 32)
    for n, k, group, text in ((0, 64, 32, "positive"), (4, 12, 32, "multiple of 8"), (4, 0, 32, "multiple of 8"),
                              (4, 64, 16, "group"), (1 << 31, 64, 32, "2\\^31")):
        with pytest.raises(ValueError, match=text):
            check(lib.msb_w4_packed_bytes(n, k, group, ctypes.byref(a), ctypes.byref(b)))
        with pytest.raises(ValueError, match=text):
            check(lib.msb_w4_product_device(_PTR, _PTR, n, k, group, _PTR, k, 1, None, _PTR, n, _lib.TYPE_F16, 0, None))
    with pytest.raises(ValueError, match="NULL"):
        check(lib.msb_w4_product_device(_PTR, None, 16, 64, 32, _PTR, 64, 1, None, _PTR, 16, _lib.TYPE_F16, 0, None))
    with pytest.raises(ValueError, match="fp16 or bf16"):
        check(lib.msb_w4_product_device(_PTR, _PTR, 16, 64, 32, _PTR, 64, 1, None, _PTR, 16, _lib.TYPE_F32, 0, None))
    for x, stride in ((_PTR + 2, 64), (_PTR, 68)):
        with pytest.raises(ValueError, match="16-byte"):
            check(lib.msb_w4_product_device(_PTR, _PTR, 16, 64, 32, x, stride, 1, None, _PTR, 16, _lib.TYPE_F16, 0, None))
    check(lib.msb_w4_product_device(None, None, 16, 64, 32, None, 64, 0, None, None, 16, _lib.TYPE_F16, 0, None))


def test_engine_option():
    assert _lib.get_option("kv4_engine") == 0
    try:
        for v in (1, 2, 0):
            _lib.set_option("kv4_engine", v)
            assert _lib.get_option("kv4_engine") == v
        with pytest.raises(ValueError, match="kv4_engine must be"):
            _lib.set_option("kv4_engine", 3)
    finally:
        _lib.set_option("kv4_engine", 0)


def test_package_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    import maxsim_b200 as m

    with pytest.raises(ValueError, match="CUDA"):
        m.Int4KVCache(2, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        m.Int4Linear(torch.zeros((4, 32), dtype=torch.uint8), torch.ones((4, 1), dtype=torch.bfloat16))
