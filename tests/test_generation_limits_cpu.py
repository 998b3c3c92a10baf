"""The cache's and the weights' host side where its arguments reach a limit: no device needed."""

import pytest

torch = pytest.importorskip("torch")

import maxsim_b200 as m  # noqa: E402


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
