"""The cache's and the weights' host side where its arguments reach a limit: no device needed."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

import maxsim_b200 as m  # noqa: E402
from maxsim_b200 import _lib  # noqa: E402
from maxsim_b200._lib import check, lib  # noqa: E402
from test_generation_cpu import _PTR, _append, _args, _cache as _c_cache  # noqa: E402


def _cache(page_size):
    """A cache's addressing alone."""
    cache = m.Int4KVCache.__new__(m.Int4KVCache)
    cache.page_size = page_size
    return cache


def test_slots_of_positions_and_of_none():
    """A slot for each position that the table holds; -1, which append skips, for every other: negative positions
    (padding), positions past the table, sequences that do not exist, entries without a page."""
    table = torch.tensor([[3, 0, -1], [5, 1 << 30, 2]], dtype=torch.int32)
    cache = _cache(16)
    for kind in (torch.int64, torch.int32):
        sequences = torch.tensor([0, 0, 0, 1, 1, 1], dtype=kind)
        positions = torch.tensor([0, 15, 16, 5, 47, 17], dtype=kind)
        got = cache.slots(table, sequences, positions)
        assert got.dtype == torch.int64 and got.tolist() == [48, 63, 0, 85, 47, (1 << 34) + 1]
        sequences = torch.tensor([0, 0, 0, 1, 1, 2, -1, -3, 0], dtype=kind)
        positions = torch.tensor([-1, -16, 48, 1 << 20, -(1 << 30), 0, 0, 5, 40], dtype=kind)
        assert cache.slots(table, sequences, positions).tolist() == [-1] * 9
    two = cache.slots(table, torch.tensor([[0], [1]]).expand(2, 3), torch.tensor([[0, -1, 18], [32, 48, 1]]))
    assert two.tolist() == [[48, -1, 2], [32, -1, 81]]


@pytest.mark.parametrize("shape", [(2, 0), (0, 3), (0, 0)])
def test_slots_of_an_empty_table(shape):
    table = torch.zeros(shape, dtype=torch.int32)
    assert _cache(64).slots(table, torch.tensor([0, 1]), torch.tensor([0, 7])).tolist() == [-1, -1]
    assert _cache(64).slots(table, torch.zeros(0, dtype=torch.int64), torch.zeros(0, dtype=torch.int64)).tolist() == []


@pytest.mark.parametrize("kw,text", [(dict(workspace=_PTR + 8, workspace_bytes=1 << 30), "workspace must be 16-byte"),
                                     (dict(workspace=None, workspace_bytes=1 << 30), "workspace is NULL"),
                                     (dict(query=_PTR + 1), "query must be 2-byte"), (dict(out=_PTR + 1), "out must be 2-byte"),
                                     (dict(page_table=_PTR + 2), "page_table must be 4-byte"),
                                     (dict(lengths=_PTR + 1), "lengths must be 4-byte"),
                                     (dict(query_offsets=_PTR + 2), "query_offsets must be 4-byte"),
                                     (dict(lse=_PTR + 2), "lse must be 4-byte")])
def test_attention_refuses_addresses_its_kernels_cannot_use(kw, text):
    with pytest.raises(ValueError, match=text):
        check(lib.msb_kv4_attend_device(ctypes.byref(_c_cache()), ctypes.byref(_args(**kw)), None))


def test_the_other_entries_refuse_addresses_their_kernels_cannot_use():
    for kw, text in ((dict(keys=_PTR + 2), "keys must be 4-byte"), (dict(values=_PTR + 1, type=_lib.TYPE_BF16), "values must be 2-byte"),
                     (dict(slots=_PTR + 4), "slots must be 8-byte")):
        with pytest.raises(ValueError, match=text):
            check(_append(_c_cache(), **kw))
    with pytest.raises(ValueError, match="slots must be 8-byte"):
        check(lib.msb_kv4_read_device(ctypes.byref(_c_cache()), _PTR + 4, 1, _lib.TYPE_BF16, _PTR, _PTR, None))

    def pack(codes=_PTR, scales=_PTR, to_codes=_PTR, to_scales=_PTR):
        check(lib.msb_w4_pack_device(codes, scales, 16, 64, 32, to_codes, to_scales, None))

    def product(codes=_PTR, scales=_PTR, bias=None, y=_PTR):
        check(lib.msb_w4_product_device(codes, scales, 16, 64, 32, _PTR, 64, 1, bias, y, 16, _lib.TYPE_F16, 0, None))

    for call, kw, text in ((pack, dict(scales=_PTR + 1), "scales must be 2-byte"), (pack, dict(to_codes=_PTR + 4), "packed_codes must be 16-byte"),
                           (pack, dict(to_scales=_PTR + 2), "packed_scales must be 4-byte"),
                           (product, dict(codes=_PTR + 8), "packed_codes must be 16-byte"),
                           (product, dict(scales=_PTR + 2), "packed_scales must be 4-byte"),
                           (product, dict(bias=_PTR + 1), "bias must be 2-byte"), (product, dict(y=_PTR + 1), "y must be 2-byte")):
        with pytest.raises(ValueError, match=text):
            call(**kw)


def test_arrays_whose_addresses_are_held_cannot_be_exchanged():
    """The kernels read the arrays that an object was made with: assigning another would leave them reading freed memory."""
    cache, linear = m.Int4KVCache.__new__(m.Int4KVCache), m.Int4Linear.__new__(m.Int4Linear)
    for thing, names in ((cache, ("k_codes", "k_scales", "v_codes", "v_scales")), (linear, ("bias",))):
        for name in names:
            with pytest.raises(AttributeError):
                setattr(thing, name, torch.zeros(1))
            with pytest.raises(AttributeError):
                delattr(thing, name)
