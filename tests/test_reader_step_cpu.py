"""Argument checks of the C entry points for masked attention, drafted trees, moves, page tables and rotary positions:
refused before any device work.  And the structs' layouts against the header."""

import ctypes
import subprocess
from pathlib import Path

import pytest

from maxsim_b200 import _lib
from maxsim_b200._lib import check, lib

REPO = Path(__file__).resolve().parent.parent
_PTR = 1 << 20  # never dereferenced: every call here is refused or has nothing to do


def _cache(**kw):
    c = dict(k_codes=_PTR, k_scales=_PTR, v_codes=_PTR, v_scales=_PTR, num_pages=4, page_size=16, kv_heads=2,
             head_dim=128, device=0)
    c.update(kw)
    return _lib.Kv4Cache(**c)


def _args(**kw):
    a = dict(query=_PTR, query_row_stride=512, query_head_stride=128, rows=2, page_table=_PTR, page_table_stride=3,
             lengths=_PTR, query_offsets=_PTR, out=_PTR, lse=None, workspace=None, workspace_bytes=0, batch=2,
             max_pages=3, max_query_rows=1, heads=4, type=_lib.TYPE_F16, causal=1, window=8, scale=0.1)
    a.update(kw)
    return _lib.Kv4AttendArgs(**a)


def _mask(**kw):
    m = dict(ancestors=_PTR, ancestors_stride=1, ancestor_words=1, sinks=4)
    m.update(kw)
    return _lib.Kv4AttendMask(**m)


@pytest.mark.parametrize("args,mask,text", [
    ({}, dict(sinks=-1), "sinks must not"), (dict(window=0), {}, "sinks need a window"),
    (dict(window=0, causal=0), dict(sinks=0), "ancestors need causal"),
    (dict(query_offsets=None), {}, "ancestors need"), ({}, dict(ancestor_words=0), "words"),
    ({}, dict(ancestor_words=1 << 25), "words"), ({}, dict(ancestors=_PTR + 4), "aligned"),
    (dict(rows=(1 << 31) - 65535, heads=1), {}, "multiple"), (dict(query=None), {}, "NULL"), (dict(rows=-1), {}, "negative")])
def test_masked_attention(args, mask, text):
    n = ctypes.c_int64()
    c, a, k = _cache(), _args(**args), _mask(**mask)
    with pytest.raises(ValueError, match=text):
        check(lib.msb_kv4_attend_masked_device(ctypes.byref(c), ctypes.byref(a), ctypes.byref(k), 0, None))
    if "NULL" not in text:
        with pytest.raises(ValueError, match=text):
            check(lib.msb_kv4_attend_masked_workspace_bytes(ctypes.byref(c), ctypes.byref(a), ctypes.byref(k), ctypes.byref(n)))


def test_rows_of_a_tree_leave_room_in_32_bits():
    c = _cache(kv_heads=1)
    a = _args(rows=(1 << 31) - 65535, heads=1)
    with pytest.raises(ValueError, match="65536 with ancestors"):
        check(lib.msb_kv4_attend_masked_device(ctypes.byref(c), ctypes.byref(a), ctypes.byref(_mask()), 0, None))


def test_masked_attention_with_nothing_to_do():
    a = _args(rows=0, batch=0, query=None, out=None, max_query_rows=0)
    check(lib.msb_kv4_attend_masked_device(ctypes.byref(_cache()), ctypes.byref(a), ctypes.byref(_mask()), 1, None))
    check(lib.msb_kv4_attend_masked_device(ctypes.byref(_cache()), ctypes.byref(a), None, 1, None))


@pytest.mark.parametrize("kw,text", [(dict(rows=-1), "negative"), (dict(batch=-1), "negative"), (dict(most=-1), "negative"),
                                     (dict(most=1025, words=17), "1024"), (dict(most=65, words=1), "words"),
                                     (dict(words=0, most=0), "words"), (dict(rows=1 << 31), "2\\^31"),
                                     (dict(parents=None), "NULL"), (dict(offsets=None), "NULL"), (dict(depths=None), "NULL"),
                                     (dict(ancestors=_PTR + 4), "aligned"), (dict(parents=_PTR + 2), "aligned")])
def test_draft_ancestors(kw, text):
    a = dict(parents=_PTR, rows=5, offsets=_PTR, batch=2, most=3, words=1, ancestors=_PTR, depths=_PTR)
    a.update(kw)
    with pytest.raises(ValueError, match=text):
        check(lib.msb_draft_ancestors_device(a["parents"], a["rows"], a["offsets"], a["batch"], a["most"], a["words"],
                                             a["ancestors"], a["depths"], 0, None))


def test_draft_ancestors_with_nothing_to_do():
    check(lib.msb_draft_ancestors_device(None, 0, None, 0, 0, 1, None, None, 0, None))


def test_move():
    n = ctypes.c_int64(7)
    check(lib.msb_kv4_move_workspace_bytes(ctypes.byref(_cache()), 1024, ctypes.byref(n)))
    assert n.value == 0
    check(lib.msb_kv4_move_workspace_bytes(ctypes.byref(_cache()), 1025, ctypes.byref(n)))
    assert n.value == 2 * 2 * 1025 * (64 + 4)
    for source, target, tokens, workspace, size, text in (
            (None, _PTR, 3, None, 0, "NULL"), (_PTR, None, 3, None, 0, "NULL"), (_PTR, _PTR, -1, None, 0, "tokens"),
            (_PTR, _PTR, 1 << 31, None, 0, "tokens"), (_PTR + 4, _PTR, 3, None, 0, "aligned"),
            (_PTR, _PTR, 1025, None, 0, "too small"), (_PTR, _PTR, 1025, None, n.value, "workspace is NULL"),
            (_PTR, _PTR, 1025, _PTR, n.value - 1, "too small"), (_PTR, _PTR, 1025, _PTR + 8, n.value, "aligned")):
        with pytest.raises(ValueError, match=text):
            check(lib.msb_kv4_move_device(ctypes.byref(_cache()), source, target, tokens, workspace, size, None))
    check(lib.msb_kv4_move_device(ctypes.byref(_cache()), None, None, 0, None, 0, None))
    with pytest.raises(ValueError, match="head_dim"):
        check(lib.msb_kv4_move_device(ctypes.byref(_cache(head_dim=96)), _PTR, _PTR, 1, None, 0, None))


def _pages(**kw):
    p = dict(page_table=_PTR, lengths=_PTR, free_pages=_PTR, free_count=_PTR, num_pages=8, sequences=2, max_pages=4,
             page_size=16, device=0)
    p.update(kw)
    return _lib.PageTableArrays(**p)


@pytest.mark.parametrize("kw,text", [(dict(page_table=None), "NULL"), (dict(free_count=None), "NULL"),
                                     (dict(lengths=_PTR + 2), "aligned"), (dict(num_pages=0), "num_pages"),
                                     (dict(num_pages=1 << 31), "num_pages"), (dict(sequences=0), "positive"),
                                     (dict(max_pages=0), "positive"), (dict(page_size=8), "page_size"),
                                     (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"),
                                     (dict(max_pages=(1 << 27) - 4095), "max_pages")])
def test_page_table_is_checked_by_every_entry_point(kw, text):
    p, n = _pages(**kw), ctypes.c_int64()
    for status in (lib.msb_pages_workspace_bytes(ctypes.byref(p), 1, ctypes.byref(n)),
                   lib.msb_pages_extend_device(ctypes.byref(p), _PTR, 1, _PTR, _PTR, _PTR, None, 0, None),
                   lib.msb_pages_truncate_device(ctypes.byref(p), _PTR, None, 0, None)):
        with pytest.raises(ValueError, match=text):
            check(status)


def test_extend_and_truncate():
    p, n = _pages(), ctypes.c_int64()
    for tokens, rows, offsets, slots, positions, text in (
            (None, 1, _PTR, _PTR, _PTR, "NULL"), (_PTR, 1, None, _PTR, _PTR, "NULL"), (_PTR, 1, _PTR, None, _PTR, "NULL"),
            (_PTR, -1, _PTR, _PTR, _PTR, "rows"), (_PTR, 1 << 31, _PTR, _PTR, _PTR, "rows"),
            (_PTR, 1, _PTR, _PTR + 4, _PTR, "aligned"), (_PTR, 1 << 20, _PTR, _PTR, _PTR, "too small")):
        with pytest.raises(ValueError, match=text):
            check(lib.msb_pages_extend_device(ctypes.byref(p), tokens, rows, offsets, slots, positions, None, 0, None))
    with pytest.raises(ValueError, match="NULL"):
        check(lib.msb_pages_truncate_device(ctypes.byref(p), None, None, 0, None))
    with pytest.raises(ValueError, match="too small"):
        check(lib.msb_pages_truncate_device(ctypes.byref(_pages(sequences=5000)), _PTR, None, 0, None))
    check(lib.msb_pages_workspace_bytes(ctypes.byref(_pages(sequences=5000)), 0, ctypes.byref(n)))
    assert n.value >= 5000 * 16


def _rotary(**kw):
    r = dict(turns=_PTR, axes=_PTR, pairs=32, head_dim=64, neighbours=0, device=0)
    r.update(kw)
    return _lib.RotaryTable(**r)


def _rotate(x=(_PTR, _PTR), y=(_PTR, _PTR), heads=(2, 1), **kw):
    a = dict(positions=_PTR, position_axis_stride=0, position_token_stride=1, tokens=3, wide_positions=0, inverse=0,
             type=_lib.TYPE_BF16)
    a.update(kw)
    strides = (ctypes.c_int64 * 2)(192, 192)
    return _lib.RotateArgs(x=(ctypes.c_void_p * 2)(*x), y=(ctypes.c_void_p * 2)(*y), x_token_stride=strides,
                           x_head_stride=strides, y_token_stride=strides, y_head_stride=strides,
                           heads=(ctypes.c_int32 * 2)(*heads), **a)


@pytest.mark.parametrize("rotary,args,text", [
    (dict(pairs=0), {}, "pairs"), (dict(pairs=33), {}, "pairs"), (dict(head_dim=0), {}, "head_dim"),
    (dict(head_dim=1026, pairs=1), {}, "head_dim"), (dict(turns=None), {}, "NULL"), (dict(axes=None), {}, "NULL"),
    (dict(turns=_PTR + 4), {}, "aligned"), ({}, dict(tokens=-1), "tokens"), ({}, dict(tokens=1 << 31), "tokens"),
    ({}, dict(heads=(-1, 1)), "heads"), ({}, dict(heads=(70000, 1)), "heads"), ({}, dict(type=7), "type must be"),
    ({}, dict(x=(None, _PTR)), "NULL"), ({}, dict(y=(_PTR, None)), "NULL"), ({}, dict(positions=None), "NULL"),
    ({}, dict(x=(_PTR + 1, _PTR)), "aligned"), ({}, dict(positions=_PTR + 2), "aligned"),
    ({}, dict(positions=_PTR + 4, wide_positions=1), "aligned")])
def test_rotate(rotary, args, text):
    with pytest.raises(ValueError, match=text):
        check(lib.msb_rotate_device(ctypes.byref(_rotary(**rotary)), ctypes.byref(_rotate(**args)), None))


def test_rotate_with_nothing_to_do():
    check(lib.msb_rotate_device(ctypes.byref(_rotary()), ctypes.byref(_rotate(tokens=0, x=(None, None), positions=None)), None))
    check(lib.msb_rotate_device(ctypes.byref(_rotary()), ctypes.byref(_rotate(heads=(0, 0), x=(None, None))), None))


def test_structs_match_the_header(tmp_path):
    pairs = {"msb_kv4_attend_mask": _lib.Kv4AttendMask, "msb_page_table": _lib.PageTableArrays, "msb_rotary": _lib.RotaryTable,
             "msb_rotate_args": _lib.RotateArgs, "msb_kv4_attend_args": _lib.Kv4AttendArgs, "msb_kv4_cache": _lib.Kv4Cache}
    body = ["#include <stdio.h>", "#include <stddef.h>", '#include "maxsim_b200.h"', "int main(void){"]
    want = []
    for name, cls in pairs.items():
        body.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, *_ in cls._fields_:
            body.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    (tmp_path / "layout.c").write_text("\n".join(body + ["return 0;}"]))
    subprocess.run(["gcc", f"-I{REPO / 'include'}", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == want


def test_package_refuses_host_devices_and_bad_sizes():
    torch = pytest.importorskip("torch")
    import maxsim_b200 as m

    for kw, text in ((dict(device="cpu"), "CUDA"), (dict(page_size=24), "page_size"), (dict(num_pages=0), "positive"),
                     (dict(max_pages=0), "positive")):
        a = dict(num_pages=4, page_size=16, max_sequences=2, max_pages=2)
        a.update(kw)
        with pytest.raises(ValueError, match=text):
            m.PageTable(**a)
    table, one = torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        m.PageTable.from_tensors(table, one, one, one[:1], page_size=16)
    for kw, text in ((dict(device="cpu"), "CUDA"), (dict(head_dim=1), "head_dim"), (dict(head_dim=2000), "head_dim"),
                     (dict(rotary_dim=66), "rotary_dim"), (dict(rotary_dim=33), "rotary_dim"), (dict(rotary_dim=0), "rotary_dim"),
                     (dict(pairs="both"), "pairs"), (dict(sections=[16, 15]), "sections"), (dict(sections=[33, -1]), "sections"),
                     (dict(sections=[]), "sections"), (dict(theta=0.0), "theta"), (dict(theta=float("inf")), "theta"),
                     (dict(frequencies=[1.0]), "frequencies"), (dict(frequencies=[float("nan")] * 32), "frequencies"),
                     (dict(sections=[8, 8, 16], interleaved=True), "interleaved")):
        a = dict(head_dim=64)
        a.update(kw)
        with pytest.raises(ValueError, match=text):
            m.Rotary(**a)
    with pytest.raises(ValueError, match="CUDA"):
        m.draft_ancestors(one, one)
    with pytest.raises(TypeError, match="tensor"):
        m.draft_ancestors([0], one)


@pytest.mark.parametrize("ancestors,depths,text", [(None, _PTR, "NULL"), (_PTR, None, "NULL"), (_PTR + 4, _PTR, "aligned")])
def test_draft_ancestors_without_sequences_still_writes(ancestors, depths, text):
    """Rows that no sequence owns are cleared, so their arrays have to be there; parents and offsets need not."""
    with pytest.raises(ValueError, match=text):
        check(lib.msb_draft_ancestors_device(None, 5, None, 0, 3, 1, ancestors, depths, 0, None))
