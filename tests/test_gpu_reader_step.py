"""What a reader model's serving step needs around its 4-bit cache, against plain arithmetic in 64 bits: attention with
sinks, trees of drafted tokens, page tables, rotary positions, moved tokens."""

import math
import random
import sys
from pathlib import Path

import numpy as np
import pytest

import maxsim_b200 as m
from maxsim_b200 import _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

sys.path.insert(0, str(Path(__file__).resolve().parent))

from test_gpu_kv4 import DTYPES, _normal, _random_cache, _tables, _values  # noqa: E402


@pytest.fixture(params=[1, 2], ids=["few", "many"])
def engine(request):
    """The attention kernel: that for few rows, that for many."""
    _lib.set_option("kv4_engine", request.param)
    yield request.param
    _lib.set_option("kv4_engine", 0)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# --------------------------------------------------------------------------- attention

def _seen(length, rows, window=None, sinks=0, parents=None):
    """[rows, length] truth values, row by row from the definition."""
    first = length - rows
    seen = torch.zeros((rows, max(length, 0)), dtype=torch.bool)
    for i in range(rows):
        if parents is None:
            p = first + i
            for j in range(0, p + 1):
                seen[i, j] = window is None or j > p - window or j < sinks
            continue
        path, at = [], i
        while at >= 0:
            path.append(at)
            at = parents[at] if 0 <= parents[at] < at else -1
        for j in range(0, first):
            seen[i, j] = window is None or j >= first + len(path) - window or j < sinks
        for a in path:
            if first + a >= 0:
                seen[i, first + a] = True
    return seen


def _check_rows(got, lse, query, cache, table, lengths, offsets, masks, scale):
    """Against the softmax in 64 bits over what `masks` let each row see.

    With p the weights (sum 1) and |v| their values' sizes: the output is rounded once (half a step of its type, relative);
    each p v is rounded to 11 bits (half a step 2^-11, relative) by the kernel, its fp32 exponential is off by 2^-21 and
    sums in fp32 add as much again, together below 2^-10 of sum p |v|; a score that is off by d moves weights by e^d, and
    so the output by 2 d sum p |v|.  Products of a score are exact, its partial sums stay below 80 sum|q| ks and are rounded
    (or cut) to 24 bits at most dim / 16 + 16 times."""
    rows, heads, dim = query.shape
    shared, page = heads // cache.num_kv_heads, cache.page_size
    step = torch.finfo(got.dtype).eps / 2
    for b, length in enumerate(lengths):
        lo, hi = offsets[b], offsets[b + 1]
        if hi == lo:
            continue
        seen = masks[b].cuda().unsqueeze(1)
        if length == 0 or not masks[b].any():
            assert not got[lo:hi].any() and torch.isinf(lse[lo:hi]).all() and (lse[lo:hi] < 0).all()
            continue
        j = torch.arange(length, device="cuda")
        pages = table[b].long()[j // page].clamp(0, cache.num_pages - 1)
        for h in range(cache.num_kv_heads):
            k = _values(cache.k_codes[pages, h, j % page], cache.k_scales[pages, h, j % page])
            v = _values(cache.v_codes[pages, h, j % page], cache.v_scales[pages, h, j % page])
            at = slice(lo, hi), slice(h * shared, (h + 1) * shared)
            q = query[at].double()
            s = (torch.einsum("nsd,jd->nsj", q, k) * scale).masked_fill(~seen, -torch.inf)
            some = seen.any(-1)
            top = torch.logsumexp(s, -1)
            p = torch.where(some.unsqueeze(-1), torch.exp(s - top.unsqueeze(-1)), 0.0)
            want = torch.einsum("nsj,jd->nsd", p, v)
            ks = torch.where(seen.any(0).any(0), cache.k_scales[pages, h, j % page].double(), 0.0).max()
            d = (q.abs().sum(-1) * ks * scale * 80 * (dim / 16 + 16) * 2.0**-23).unsqueeze(-1)
            limit = step * want.abs() + (2.0**-10 + 2 * d) * torch.einsum("nsj,jd->nsd", p, v.abs()) + 1e-30
            off = (got[at].double() - want).abs()
            assert (off <= limit).all(), f"sequence {b}, head {h}: {(off / limit).max().item():.3g} of the bound"
            assert torch.equal(torch.isinf(lse[at]), ~some.expand(-1, shared))
            held = some.expand(-1, shared)
            assert ((lse[at].double() - top).abs() <= d.squeeze(-1) + 1e-5 + 1e-6 * top.abs())[held].all()


def _run(dim, heads, shared, page, dtype, lengths, rows=None, window=None, sinks=0, trees=None, seed=0):
    """One call, checked; `trees`: each sequence's parents."""
    pages = sum(-(-n // page) for n in lengths) + 2
    cache = _random_cache(pages, page, heads, dim, seed)
    table = _tables(lengths, page, pages, seed=seed)
    count = [1] * len(lengths) if rows is None else rows
    offsets = [0] + np.cumsum(count).tolist()
    query = _normal((offsets[-1], heads * shared, dim), seed + 9, DTYPES[dtype], 1.5)
    starts = None if rows is None else _int32(offsets)
    most = None if rows is None else max(rows)
    ancestors = None
    if trees is not None:
        ancestors, depths = m.draft_ancestors(_int32([p for t in trees for p in t]), starts, max_query_tokens=most)
    got, lse = cache.attend(query, table, _int32(lengths), query_offsets=starts, max_query_tokens=most, window=window,
                            sinks=sinks, ancestors=ancestors, return_lse=True)
    masks = [_seen(n, r, window, sinks, None if trees is None else trees[b]) for b, (n, r) in enumerate(zip(lengths, count))]
    _check_rows(got, lse, query, cache, table, lengths, offsets, masks, dim**-0.5)
    return cache, table, query, starts, most, ancestors, got, masks


def _tree(rows, seed, reach=8):
    rng = random.Random(seed)
    return [rng.randint(max(-1, i - reach), i - 1) for i in range(rows)]


@pytest.mark.parametrize("dtype,dim", [("f16", 64), ("bf16", 128), ("bf16", 256)])
@pytest.mark.parametrize("window", [1, 33, 200])
@pytest.mark.parametrize("sinks", [1, 31, 32, 33, 129, 1000])
def test_sinks_of_one_token(dtype, dim, window, sinks):
    """Lengths where the window has not left the sinks, touches them, or is far past them; an empty sequence."""
    _run(dim, 2, 4, 16, dtype, [0, 1, 2, 33, 64, 129, 200, 201, 233, 330, 1030], window=window, sinks=sinks, seed=sinks)


@pytest.mark.parametrize("dim,shared", [(64, 1), (128, 4), (128, 9), (256, 2)])
@pytest.mark.parametrize("window,sinks", [(1, 1), (33, 4), (100, 128), (130, 300), (1000, 7)])
def test_sinks_of_ragged_rows(engine, dim, shared, window, sinks):
    """Several rows a sequence, some without rows, one with more rows than tokens."""
    _run(dim, 2, shared, 32, "bf16", [5, 70, 0, 530, 64, 3, 1257], rows=[5, 1, 3, 40, 0, 7, 129], window=window, sinks=sinks,
         seed=shared)


@pytest.mark.parametrize("page", [16, 64, 1024])
def test_sinks_of_long_contexts(page):
    """Ranges of the work line that end within the sinks, the gap's edges, the window."""
    _run(128, 8, 4, page, "f16", [20000, 7000, 3001, 15, 0], window=2500, sinks=700, seed=page)


@pytest.mark.parametrize("batch", [1, 31, 40, 200])
def test_sinks_of_many_sequences(batch):
    _run(64, 1, 2, 16, "bf16", [(37 * b) % 900 for b in range(batch)], window=100, sinks=20, seed=batch)


@pytest.mark.parametrize("batch,heads,long", [(300, 8, 0), (700, 4, 3000)])
def test_more_short_sequences_than_a_block_lists_at_once(engine, batch, heads, long):
    """Hundreds of segments of a tile for each block, and (`long`) a few of many tiles among them."""
    lengths = [long if long and b % 99 == 7 else (7 * b) % 45 for b in range(batch)]
    rows = [b % 4 for b in range(batch)]
    _run(64, heads, 2, 16, "f16", lengths, rows=rows, window=600, sinks=9, seed=batch)
    _run(64, heads, 2, 16, "f16", lengths, rows=rows, trees=[_tree(r, r) for r in rows], seed=batch)


@pytest.mark.parametrize("dtype,dim,shared", [("f16", 64, 1), ("bf16", 128, 4), ("f16", 128, 7), ("bf16", 256, 2)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (40, 3), (300, 64)])
def test_trees(engine, dtype, dim, shared, window, sinks):
    """Ragged trees, one word of masks to three; a sequence without rows, one without context, one with fewer tokens
    than rows."""
    rows = [1, 13, 0, 64, 65, 130, 20, 9]
    lengths = [500, 13, 77, 300, 1111, 700, 12, 0]
    _run(dim, 2, shared, 16, dtype, lengths, rows=rows, window=window, sinks=sinks, trees=[_tree(r, r) for r in rows], seed=shared)


@pytest.mark.parametrize("rows,length", [(1, 1), (2, 40), (31, 95), (32, 96), (33, 97), (64, 64), (64, 8000), (100, 1000)])
def test_trees_at_the_edges_of_tiles(engine, rows, length):
    _run(128, 2, 4, 64, "bf16", [length], rows=[rows], trees=[_tree(rows, length)], seed=rows)


def test_a_chain_is_what_causal_rows_see(engine):
    """A tree of one path is the same call without it, and a bit for every row is the call without causal."""
    lengths, rows = [300, 700], [40, 70]
    cache, table, query, starts, most, _, got, _ = _run(128, 2, 4, 16, "bf16", lengths, rows=rows,
                                                        trees=[list(range(-1, r - 1)) for r in rows])
    plain = cache.attend(query, table, _int32(lengths), query_offsets=starts, max_query_tokens=most)
    # Both are off by half a step at most from sums that differ by less.
    assert ((got.double() - plain.double()).abs() <= 2.0**-7 * plain.double().abs() + 2.0**-9 * 3).all()
    every = torch.full((sum(rows), 2), -1, dtype=torch.int64, device="cuda")
    seen = cache.attend(query, table, _int32(lengths), query_offsets=starts, max_query_tokens=most, ancestors=every, return_lse=True)
    masks = [torch.ones((r, n), dtype=torch.bool) for r, n in zip(rows, lengths)]
    _check_rows(seen[0], seen[1], query, cache, table, lengths, starts.tolist(), masks, 128**-0.5)


def test_masks_that_leave_rows_empty(engine):
    """No context and no bits: zeros and -inf; bits of rows that are not there, and words past the rows, count nothing."""
    lengths, rows = [6, 0, 90], [6, 3, 4]
    cache = _random_cache(10, 16, 2, 64, 3)
    table = _tables(lengths, 16, 10)
    query = _normal((13, 4, 64), 4, torch.float16)
    starts = _int32([0, 6, 9, 13])
    bits = torch.zeros((13, 3), dtype=torch.int64, device="cuda")
    bits[1, 0] = 1 << 1
    bits[3, 0] = (1 << 2) | (1 << 6) | (1 << 40)  # rows 6 and 40 are not there
    bits[4] = -1
    bits[9:, 1:] = -1
    bits[10, 0] = -1
    got, lse = cache.attend(query, table, _int32(lengths), query_offsets=starts, max_query_tokens=6, ancestors=bits,
                            return_lse=True)
    masks = [torch.zeros((r, n), dtype=torch.bool) for r, n in zip(rows, lengths)]
    masks[0][1, 1] = masks[0][3, 2] = True
    masks[0][4] = True
    masks[2][:, :86] = True
    masks[2][1] = True
    _check_rows(got, lse, query, cache, table, lengths, [0, 6, 9, 13], masks, 64**-0.5)
    # With a window these bits take places in it: row 1 of the last sequence has four, row 0 none.
    got, lse = cache.attend(query, table, _int32(lengths), query_offsets=starts, max_query_tokens=6, ancestors=bits,
                            window=10, sinks=2, return_lse=True)
    masks[2][:] = False
    masks[2][:, :2] = True
    masks[2][:, 76:86] = True
    masks[2][1, 76:80] = False
    masks[2][1, 86:] = True
    _check_rows(got, lse, query, cache, table, lengths, [0, 6, 9, 13], masks, 64**-0.5)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_does_not_matter(engine, dim, tree):
    """NaN, infinite and huge scales in every slot that no row sees (the gap, other branches, the rest of a page) leave
    the results bit for bit the same."""
    lengths, rows, page = [400, 16, 1000], [7, 1, 50], 16
    trees = [[-1] * r for r in rows] if tree else None  # every node by itself: a row's neighbours are not seen
    cache, table, query, starts, most, bits, got, masks = _run(dim, 2, 4, page, "f16", lengths, rows=rows, window=50, sinks=5,
                                                               trees=trees, seed=4)
    used = torch.zeros((cache.num_pages, page), dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        j = masks[b].any(0).nonzero().squeeze(1).cuda()
        used[table[b].long()[j // page], j % page] = True
    for bad in (float("nan"), float("inf"), 3e38, -float("inf")):
        for t in (cache.k_scales, cache.v_scales):
            t.copy_(torch.where(used.unsqueeze(1), t, bad))
        again = cache.attend(query, table, _int32(lengths), query_offsets=starts, max_query_tokens=most, window=50, sinks=5,
                             ancestors=bits)
        assert torch.equal(got, again)


def test_another_branch_that_is_not_finite(engine):
    """A node with a NaN harms the rows below it alone."""
    parents = [-1, 0, 0, 1, 2, 3, 4]
    cache = _random_cache(4, 16, 1, 128, seed=6)
    table, lengths, starts = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), _int32([57]), _int32([0, 7])
    bits, _ = m.draft_ancestors(_int32(parents), starts)
    q = _normal((7, 4, 128), 1, torch.bfloat16)
    clean = cache.attend(q, table, lengths, query_offsets=starts, max_query_tokens=7, ancestors=bits)
    cache.v_scales[51 // 16, 0, 51 % 16] = float("nan")  # row 1, above 3 and 5
    got = cache.attend(q, table, lengths, query_offsets=starts, max_query_tokens=7, ancestors=bits)
    for i in range(7):
        if i in (1, 3, 5):
            assert torch.isnan(got[i]).all()
        else:
            assert torch.equal(got[i], clean[i])


def test_pages_before_the_window_may_be_gone(engine):
    """Table entries between the sinks and the window that name no page of the cache change nothing."""
    lengths = [900, 1500]
    cache, table, query, starts, most, _, got, _ = _run(128, 2, 4, 16, "bf16", lengths, rows=[3, 1], window=128, sinks=16)
    gone = table.clone()
    gone[0, 1:(897 - 128) // 16] = -1
    gone[1, 1:(1499 - 128) // 16] = 1 << 30
    again = cache.attend(query, gone, _int32(lengths), query_offsets=starts, max_query_tokens=most, window=128, sinks=16)
    assert torch.equal(got, again)


def test_windows_and_sinks_near_2_to_31(engine):
    """A window larger than any length: sinks change nothing; sinks larger than any length: the window changes nothing."""
    lengths, rows = [300, 7], [20, 9]
    cache, table, query, starts, most, _, got, _ = _run(64, 2, 4, 16, "f16", lengths, rows=rows)
    for window, sinks in ((2**31 - 1, 2**31 - 1), (2**40, 3), (1, 2**31 - 1), (1, 2**40)):
        again = cache.attend(query, table, _int32(lengths), query_offsets=starts, max_query_tokens=most, window=window, sinks=sinks)
        assert ((again.double() - got.double()).abs() <= 2.0**-9 * got.double().abs() + 2.0**-9 * 3).all()
    bits, _ = m.draft_ancestors(_int32(list(range(-1, 19)) + list(range(-1, 8))), starts, max_query_tokens=20)
    for window, sinks in ((2**31 - 1, 0), (2**31 - 1, 2**31 - 1)):
        again = cache.attend(query, table, _int32(lengths), query_offsets=starts, max_query_tokens=most, window=window,
                             sinks=sinks, ancestors=bits)
        assert ((again.double() - got.double()).abs() <= 2.0**-9 * got.double().abs() + 2.0**-9 * 3).all()


def test_rows_without_a_sequence_and_rows_past_the_announced(engine):
    """Padding is zero, rows past `max_query_tokens` NaN, as without masks; the others see what they saw."""
    lengths, rows = [300, 500], [5, 9]
    cache, table, query, starts, most, bits, got, _ = _run(64, 2, 4, 16, "f16", lengths, rows=rows, trees=[_tree(r, r) for r in rows])
    wide = torch.cat((query[:3], query, query[:2]))
    shifted = starts + 3
    masks = torch.cat((bits[:3], bits, bits[:2]))
    padded = cache.attend(wide, table, _int32(lengths), query_offsets=shifted, max_query_tokens=9, ancestors=masks)
    assert torch.equal(padded[3:17], got) and not padded[:3].any() and not padded[17:].any()
    few = cache.attend(wide, table, _int32(lengths), query_offsets=shifted, max_query_tokens=6, ancestors=masks)
    assert torch.equal(few[3:14], got[:11]) and torch.isnan(few[14:17]).all()
    out = torch.full_like(wide, 7.0)
    cache.attend(wide, table, _int32(lengths), query_offsets=shifted, max_query_tokens=9, ancestors=masks, out=out)
    assert torch.equal(out[3:17], got) and (out[:3] == 7).all() and (out[17:] == 7).all()


def test_strided_masks_and_results_that_repeat(engine):
    lengths, rows = [300, 2000], [70, 90]
    cache, table, query, starts, most, bits, got, _ = _run(128, 2, 2, 16, "bf16", lengths, rows=rows, window=500, sinks=40,
                                                           trees=[_tree(r, r) for r in rows])
    spread = torch.full((160, 7), -1, dtype=torch.int64, device="cuda")
    spread[:, 2:4] = bits
    every_other = torch.full((160, 4), -1, dtype=torch.int64, device="cuda")
    every_other[:, ::2] = bits
    for b in (bits, spread[:, 2:4], every_other[:, ::2]):
        again = cache.attend(query, table, _int32(lengths), query_offsets=starts, max_query_tokens=most, window=500, sinks=40,
                             ancestors=b)
        assert torch.equal(got, again)


def test_masked_attention_past_4_gb_of_codes():
    page, heads, dim = 1024, 8, 128
    pages = 9000  # 4.7 GB of codes for keys, as much for values
    cache = m.Int4KVCache(pages, page, heads, dim)
    small = m.Int4KVCache(3, page, heads, dim)
    k, v = _normal((3 * page, heads, dim), 1, torch.bfloat16), _normal((3 * page, heads, dim), 2, torch.bfloat16)
    near, far = torch.arange(3 * page, device="cuda"), torch.arange((pages - 3) * page, pages * page, device="cuda")
    small.append(k, v, near)
    cache.append(k, v, near)
    cache.move(near, far)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(far), small.read(near)))
    cache.k_codes[:3], cache.v_codes[:3] = 0, 0
    ids = torch.tensor([[pages - 3, pages - 2, pages - 1]], dtype=torch.int32, device="cuda")
    for rows in (1, 200):
        q, starts, length = _normal((rows, 16, dim), 3, torch.bfloat16), _int32([0, rows]), _int32([3 * page - 5])
        bits, _ = m.draft_ancestors(_int32(_tree(rows, rows)), starts)
        for kw in (dict(window=900, sinks=70), dict(ancestors=bits)):
            a = cache.attend(q, ids, length, query_offsets=starts, max_query_tokens=rows, **kw)
            b = small.attend(q, _int32([[0, 1, 2]]), length, query_offsets=starts, max_query_tokens=rows, **kw)
            assert torch.equal(a, b)


# --------------------------------------------------------------------------- drafted trees

def _walk(parents):
    bits, depths = [], []
    for i, p in enumerate(parents):
        up = p if 0 <= p < i else -1
        bits.append((bits[up] if up >= 0 else 0) | 1 << i)
        depths.append(depths[up] + 1 if up >= 0 else 0)
    return bits, depths


@pytest.mark.parametrize("rows,most", [([1], None), ([5, 0, 3], None), ([64, 63, 1], 64), ([65, 128, 129], 129),
                                       ([1000, 1024], 1024), ([1] * 300, 1)])
def test_draft_ancestors(rows, most):
    rng = random.Random(sum(rows))
    trees = [[rng.choice([-1, i - 1, rng.randint(-5, i + 3), i, 1 << 30, -(1 << 31)]) for i in range(r)] for r in rows]
    starts = [0] + np.cumsum(rows).tolist()
    bits, depths = m.draft_ancestors(_int32([p for t in trees for p in t]), _int32(starts), max_query_tokens=most)
    assert bits.shape == (starts[-1], -(-(most or min(1024, starts[-1])) // 64)) and bits.dtype == torch.int64
    got, at = bits.tolist(), 0
    for t in trees:
        want, want_depths = _walk(t)
        for i in range(len(t)):
            assert sum((w % 2**64) << 64 * k for k, w in enumerate(got[at + i])) == want[i]
        assert depths[at:at + len(t)].tolist() == want_depths
        at += len(t)


def test_draft_ancestors_of_padding_and_bad_offsets():
    parents = _int32([-1, 0, 1, 2, 3, 4, 5, 6, 7, 8])
    for _ in range(3):  # fresh memory that holds something
        junk = torch.full((10, 1), -1, dtype=torch.int64, device="cuda")
        del junk
        bits, depths = m.draft_ancestors(parents, _int32([2, 5, 8]), max_query_tokens=2)
        assert bits[:, 0].tolist() == [0, 0, 1, 2, 0, 1, 2, 0, 0, 0]  # a parent before its node alone counts
        assert depths.tolist() == [0] * 10
    bits, depths = m.draft_ancestors(_int32([-1, 0, 0, 2]), _int32([-7, 2, 900]), max_query_tokens=4)
    assert bits[:, 0].tolist() == [1, 3, 1, 2] and depths.tolist() == [0, 1, 0, 0]
    bits, depths = m.draft_ancestors(_int32([-1, 0, 0, 2]), _int32([0]), max_query_tokens=4)
    assert not bits.any() and not depths.any()
    bits, depths = m.draft_ancestors(_int32([]), _int32([0, 0]))
    assert bits.shape == (0, 1) and depths.shape == (0,)
    m.draft_ancestors(_int32([-1, 0, 0, 2]), _int32([5, 3, 1]), max_query_tokens=4)
    with pytest.raises(ValueError, match="1024"):
        m.draft_ancestors(torch.zeros(1025, dtype=torch.int32, device="cuda"), _int32([0, 1025]))
    for args, text in (((parents.long(), _int32([0, 1])), "dtype"), ((parents.view(2, 5), _int32([0, 1])), "dimensions"),
                       ((parents, _int32([])), "batch"), ((parents, torch.tensor([0, 1], dtype=torch.int32)), "must be on")):
        with pytest.raises(ValueError, match=text):
            m.draft_ancestors(*args)


# --------------------------------------------------------------------------- page tables

class _Pages:
    """The page table in plain Python."""

    def __init__(self, table, lengths, free, size):
        self.table, self.lengths, self.free, self.size = [list(r) for r in table], list(lengths), list(free), size

    def extend(self, tokens, rows):
        size, start, asked, out_slots, out_positions, offsets = self.size, 0, 0, [-1] * rows, [-1] * rows, [0]
        free = list(self.free)
        for b, n in enumerate(tokens):
            n = max(0, n)
            have, want = -(-self.lengths[b] // size), -(-(self.lengths[b] + n) // size)
            fits = want <= len(self.table[b]) and start + n <= rows
            lacks = want - have if fits else 0
            asked += lacks
            if fits and (lacks == 0 or asked <= len(free)):
                for c in range(have, want):
                    self.table[b][c] = self.free.pop()
                for i in range(n):
                    p = self.lengths[b] + i
                    out_positions[start + i] = p
                    out_slots[start + i] = self.table[b][p // size] * size + p % size
                self.lengths[b] += n
            start += n
            offsets.append(min(start, rows))
        return offsets, out_slots, out_positions

    def truncate(self, lengths):
        back = []
        for b, n in enumerate(lengths):
            n = min(max(0, n), self.lengths[b])
            for c in range(-(-n // self.size), -(-self.lengths[b] // self.size)):
                back.append(self.table[b][c])
                self.table[b][c] = -1
            self.lengths[b] = n
        self.free += back[::-1]


def _same(pages, plain):
    assert pages.lengths.tolist() == plain.lengths
    assert pages.free_count.item() == len(plain.free)
    assert pages.free_pages[:len(plain.free)].tolist() == plain.free
    assert pages.page_table.tolist() == plain.table


@pytest.mark.parametrize("sequences,columns,size,pages,most,steps", [
    (1, 1, 16, 1, 20, 12), (3, 4, 16, 9, 40, 30), (64, 40, 64, 900, 100, 12), (1000, 3, 16, 1500, 9, 8),
    (1025, 3, 16, 1500, 9, 8), (2500, 4, 32, 9000, 30, 5), (5, 2000, 16, 5000, 9000, 6)])
def test_page_table_against_plain_python(sequences, columns, size, pages, most, steps):
    """Random growth and shrinkage until pages, columns and rows run out; one block's sizes and several blocks'."""
    rng = random.Random(sequences)
    table = m.PageTable(pages, size, sequences, columns)
    plain = _Pages(table.page_table.tolist(), table.lengths.tolist(), table.free_pages.tolist(), size)
    for step in range(steps):
        tokens = [rng.choice([0, 1, rng.randint(-3, most)]) for _ in range(sequences)]
        total = sum(max(0, n) for n in tokens)
        rows = rng.choice([total, total + 5, max(0, total - 3)])
        got = table.extend(_int32(tokens), rows)
        for g, w, dtype in zip(got, plain.extend(tokens, rows), (torch.int32, torch.int64, torch.int32)):
            assert g.dtype == dtype and g.tolist() == w
        _same(table, plain)
        if step % 2:
            lengths = [rng.choice([n, n + 7, rng.randint(-2, n + 1), 0 if step % 4 == 3 else n]) for n in plain.lengths]
            table.truncate(_int32(lengths))
            plain.truncate(lengths)
            _same(table, plain)
    held = [p for r in plain.table for p in r if p >= 0] + plain.free
    assert sorted(held) == list(range(pages))


def test_a_step_taken_back_leaves_the_table_as_it_was():
    table = m.PageTable(200, 16, 7, 60)
    table.extend(_int32([5, 0, 100, 16, 17, 300, 1]), 439)
    before = [t.clone() for t in (table.page_table, table.lengths, table.free_pages, table.free_count)]
    table.extend(_int32([64, 3, 0, 16, 15, 33, 900]), 1031)
    table.truncate(before[1])
    for t, old in zip((table.page_table, table.lengths, table.free_pages, table.free_count), before):
        assert torch.equal(t, old)
    table.truncate(table.lengths)  # its own lengths: nothing happens
    for t, old in zip((table.page_table, table.lengths, table.free_pages, table.free_count), before):
        assert torch.equal(t, old)


def test_the_sequence_that_lacks_no_page_is_served_when_none_are_left():
    table = m.PageTable(3, 16, 4, 2)
    table.extend(_int32([10, 16, 3, 0]), 29)
    offsets, slots, positions = table.extend(_int32([6, 1, 2, 1]), 10)
    assert offsets.tolist() == [0, 6, 7, 9, 10]
    assert positions.tolist() == [10, 11, 12, 13, 14, 15, -1, 3, 4, -1]
    assert slots.tolist() == [10, 11, 12, 13, 14, 15, -1, 35, 36, -1]
    assert table.lengths.tolist() == [16, 16, 5, 0] and table.free_count.item() == 0


def test_page_tables_that_hold_nonsense_stay_in_bounds():
    """Lengths, counts and ids that no call would have left: nothing outside the arrays is read or written."""
    for sequences in (3, 1500):
        guard = torch.full((4096 + 4 * sequences,), 12345, dtype=torch.int32, device="cuda")
        arrays = (guard[1024:1024 + 4 * sequences].view(sequences, 4), torch.empty(sequences, dtype=torch.int32, device="cuda"),
                  torch.empty(6, dtype=torch.int32, device="cuda"), _int32([0]))
        for lengths, count, page in ((1 << 30, 1 << 30, -5), (-9, -9, 1 << 30), (63, 6, -(1 << 31))):
            arrays[0].fill_(page)
            arrays[1].fill_(lengths)
            arrays[2].fill_(page)
            arrays[3].fill_(count)
            table = m.PageTable.from_tensors(*arrays, page_size=16)
            tokens = torch.full((sequences,), 7, dtype=torch.int32, device="cuda")
            _, slots, positions = table.extend(tokens, 7 * sequences)
            assert ((positions >= -1) & (positions < 64)).all()
            table.truncate(torch.full((sequences,), -3, dtype=torch.int32, device="cuda"))
            assert (table.lengths == 0).all() and 0 <= table.free_count.item() <= 6
            assert (guard[:1024] == 12345).all() and (guard[1024 + 4 * sequences:] == 12345).all()


def test_page_table_refusals():
    table = m.PageTable(8, 16, 3, 4)
    good = _int32([1, 2, 3])
    for args, error, text in (((good.long(), 6), ValueError, "dtype"), ((good[:2], 6), ValueError, "shape"),
                              ((good.cpu(), 6), ValueError, "must be on"), ((good, -1), ValueError, "rows"),
                              ((good, 1 << 31), ValueError, "rows"), (([1, 2, 3], 6), TypeError, "tensor"),
                              ((table.free_pages[2:5], 6), ValueError, "overlap"), ((table.page_table[0, :3], 6), ValueError, "overlap")):
        with pytest.raises(error, match=text):
            table.extend(*args)
    with pytest.raises(ValueError, match="shape"):
        table.truncate(good[:1])
    with pytest.raises(ValueError, match="overlap"):
        table.truncate(table.page_table[1, :3])
    a = (table.page_table, table.lengths, table.free_pages, table.free_count)
    for bad, text in (((a[0].long(), *a[1:]), "dtype"), ((a[0][:, ::2], *a[1:]), "contiguous"), ((a[0], a[1][:2], *a[2:]), "shape"),
                      ((a[0], a[1], a[0].view(-1)[:8], a[3]), "overlap"), ((a[0][:0], a[1][:0], a[2], a[3]), "positive")):
        with pytest.raises(ValueError, match=text):
            m.PageTable.from_tensors(*bad, page_size=16)
    with pytest.raises(AttributeError):
        table.lengths = good


# --------------------------------------------------------------------------- rotary positions

def _angles(rotary_dim, sections, interleaved, positions, theta=10000.0, inverse=False):
    """[tokens, pairs] in 64 bits."""
    half, n = rotary_dim // 2, len(sections)
    columns = []
    for i in range(half):
        if interleaved:
            axis = i % n if i < n * sections[i % n] else 0
        else:
            axis = next(a for a in range(n) if i < sum(sections[:a + 1]))
        columns.append(positions[axis].double() * theta ** (-i / half))
    angles = torch.stack(columns, dim=1)
    return -angles if inverse else angles


def _check_turned(got, x, angles, rotary_dim, neighbours, slack=0.0):
    """|got - want| <= half a step of the output's type + 2^-22 (|a| + |b|): sines and cosines off by less than 2^-23
    (their own 2^-24, the angle's rounding 2^-25 of an eighth of a turn), one product and one sum in fp32."""
    half = rotary_dim // 2
    c, s = torch.cos(angles).unsqueeze(1), torch.sin(angles).unsqueeze(1)
    f = x.double()
    a, b = (f[..., 0:rotary_dim:2], f[..., 1:rotary_dim:2]) if neighbours else (f[..., :half], f[..., half:rotary_dim])
    g = got.double()
    ga, gb = (g[..., 0:rotary_dim:2], g[..., 1:rotary_dim:2]) if neighbours else (g[..., :half], g[..., half:rotary_dim])
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps  # the smallest number above 0
    for value, want in ((ga, a * c - b * s), (gb, a * s + b * c)):
        limit = torch.finfo(got.dtype).eps / 2 * want.abs() + (2.0**-22 + slack) * (a.abs() + b.abs()) + tiny
        assert ((value - want).abs() <= limit).all(), ((value - want).abs() / limit).max().item()
    assert torch.equal(got[..., rotary_dim:], x[..., rotary_dim:])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("dim,rotary_dim,sections,interleaved,heads,kv_heads,tokens", [
    (64, 64, [32], False, 1, 1, 1), (128, 128, [16, 24, 24], False, 32, 8, 33), (128, 128, [24, 20, 20], True, 5, 0, 100),
    (96, 48, [7, 17], False, 5, 1, 77), (80, 20, [10], False, 3, 2, 9), (256, 256, [100, 28], False, 2, 1, 515),
    (6, 2, [1], False, 1, 1, 40), (7, 6, [1, 1, 1], True, 3, 2, 65), (1024, 1024, [512], False, 3, 1, 5), (72, 64, [0, 32], False, 300, 1, 3)])
def test_rotary(dtype, pairs, dim, rotary_dim, sections, interleaved, heads, kv_heads, tokens):
    rotary = m.Rotary(dim, sections=sections, rotary_dim=rotary_dim, interleaved=interleaved, pairs=pairs)
    q = _normal((tokens, heads, dim), 1, DTYPES[dtype])
    k = _normal((tokens, kv_heads, dim), 2, DTYPES[dtype]) if kv_heads else None
    g = torch.Generator().manual_seed(tokens)
    positions = torch.randint(-50, 40000, (len(sections), tokens), generator=g).cuda()
    for inverse in (False, True):
        for p in (positions, positions.int()):
            angles = _angles(rotary_dim, sections, interleaved, positions, inverse=inverse)
            got = rotary(q, k, p, inverse=inverse)
            _check_turned(got[0], q, angles, rotary_dim, pairs == "neighbours")
            if k is None:
                assert got[1] is None
            else:
                _check_turned(got[1], k, angles, rotary_dim, pairs == "neighbours")


def test_rotary_at_far_positions():
    """Angles past 2^31 radians are as exact as near ones.  (The 64-bit angle itself is off by 2^-53 of its size.)"""
    positions = torch.tensor([0, 1, -1, 131071, 10**6, 2**31 - 1, -(2**31), 2**40, -(2**40)], device="cuda")
    rotary = m.Rotary(64, theta=500000.0)
    q = _normal((9, 3, 64), 1)
    got, _ = rotary(q, None, positions)
    angles = _angles(64, [32], False, positions.view(1, 9), theta=500000.0)
    _check_turned(got[:7], q[:7], angles[:7], 64, False, slack=2.0**31 * 2.0**-52)
    _check_turned(got, q, angles, 64, False, slack=2.0**40 * 2.0**-52)
    assert torch.equal(rotary(q[:7], None, positions[:7].int())[0], got[:7])


def test_rotary_with_frequencies_and_back():
    frequencies = [0.0, math.pi / 2, -math.pi, 3 * math.pi, 1e-9, 1e9, 0.125, 2.5]
    rotary = m.Rotary(16, frequencies=frequencies, pairs="neighbours")
    positions = torch.arange(-3, 6, dtype=torch.int32, device="cuda")
    x = _normal((9, 2, 16), 3)
    got, none = rotary(x, None, positions)
    angles = positions.double().unsqueeze(1) * torch.tensor(frequencies, dtype=torch.float64, device="cuda")
    _check_turned(got, x, angles, 16, True, slack=9e9 * 2.0**-52)
    assert torch.equal(got[..., :2], x[..., :2])  # frequency 0 turns nothing
    assert torch.equal(got[3], x[3])              # nor does position 0
    back, _ = rotary(got, None, positions, inverse=True)
    # two turns, each within 2^-22 (|a| + |b|) and a rounding
    assert ((back - x).abs() <= 2.0**-20 * (x.abs() + x.unflatten(-1, (8, 2)).flip(-1).flatten(-2).abs())).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,offset", [(128, 0), (128, 1), (64, 8), (96, 4)])
def test_rotary_strides_and_in_place(dtype, dim, offset):
    """Views of a projection's rows, heads before tokens, dimensions apart; in place and into other views: the same bits;
    what lies beside is untouched."""
    tokens, heads, kv = 37, 6, 2
    rotary = m.Rotary(dim, sections=[dim // 8, dim // 8, dim // 4])
    positions = torch.randint(0, 999, (tokens, 3), device="cuda").t()
    wide = _normal((tokens, (heads + 2 * kv) * dim + 2 * offset), 5, DTYPES[dtype])
    qkv = wide[:, offset:wide.shape[1] - offset].unflatten(1, (heads + 2 * kv, dim))
    q, k, v = qkv.split((heads, kv, kv), dim=1)
    want = rotary(q.contiguous(), k.contiguous(), positions)
    _check_turned(want[0], q, _angles(dim, [dim // 8, dim // 8, dim // 4], False, positions), dim, False)
    for a, b in ((q, k), (q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(1, 2).contiguous().transpose(1, 2))):
        got = rotary(a, b, positions)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = torch.full_like(wide, 7.0)
    oqkv = out[:, offset:wide.shape[1] - offset].unflatten(1, (heads + 2 * kv, dim))
    oq, ok, ov = oqkv.split((heads, kv, kv), dim=1)
    got = rotary(q, k, positions, out=(oq, ok))
    assert torch.equal(oq, want[0]) and torch.equal(ok, want[1]) and (ov == 7).all() and torch.equal(got[0], oq)
    if offset:
        assert (out[:, :offset] == 7).all() and (out[:, -offset:] == 7).all()
    old = v.clone()
    rotary(q, k, positions, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, old)


def test_rotary_of_values_that_are_not_finite():
    """They stay in their pair."""
    rotary = m.Rotary(64)
    x = _normal((3, 2, 64), 1, torch.bfloat16)
    y = x.clone()
    y[1, 1, 5], y[2, 0, 40] = float("nan"), float("inf")
    positions = torch.arange(3, device="cuda")
    clean, got = rotary(x, None, positions)[0], rotary(y, None, positions)[0]
    keep = torch.ones_like(x, dtype=torch.bool)
    keep[1, 1, [5, 37]] = keep[2, 0, [8, 40]] = False
    assert torch.equal(got[keep], clean[keep]) and not torch.isfinite(got[~keep]).any()


def test_rotary_refusals():
    rotary = m.Rotary(64, sections=[16, 16])
    q, k = _normal((5, 4, 64), 1, torch.bfloat16), _normal((5, 2, 64), 2, torch.bfloat16)
    p = torch.zeros((2, 5), dtype=torch.int64, device="cuda")
    for args, kw, error, text in (
            ((q[..., :32], k, p), {}, ValueError, "shape"), ((q, k.half(), p), {}, ValueError, "same dtype"),
            ((q, k[:4], p), {}, ValueError, "same number"), ((q.double(), None, p), {}, ValueError, "dtype"),
            ((q, k, p[:1]), {}, ValueError, "positions"), ((q, k, p[0]), {}, ValueError, "positions"),
            ((q, k, p[:, :4]), {}, ValueError, "same number"), ((q, k, p.float()), {}, ValueError, "positions"),
            ((q, k, p.cpu()), {}, ValueError, "must be on"), ((q.flatten(1), k, p), {}, ValueError, "dimensions"),
            ((None, k, p), {}, TypeError, "tensor"), ((q, k, p), {"out": q}, TypeError, "pair"),
            ((q, k, p), {"out": (q, None)}, TypeError, "tensor"), ((q, None, p), {"out": (q, k)}, ValueError, "None"),
            ((q, k, p), {"out": (q.half(), k)}, ValueError, "dtype"), ((q, k, p), {"out": (q[:4], k)}, ValueError, "shape"),
            ((q, k, p), {"out": (k.repeat(1, 2, 1)[:, :1].expand(5, 4, 64), k)}, ValueError, "itself"),
            ((q[:, :2], k, p), {"out": (k, q[:, :2])}, ValueError, "apart"),
            ((q[:4], k[:4], p[:, :4]), {"out": (q[1:], k[:4])}, ValueError, "apart"),
            ((q[:, :2], k, p), {"out": (q[:, 1:3], k)}, ValueError, "apart")):
        with pytest.raises(error, match=text):
            rotary(*args, **kw)
    same = torch.empty((5, 2, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="apart"):
        rotary(q[:, :2], k, p, out=(same, same))
    store = torch.zeros((5, 4, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="apart from positions"):
        rotary(q, None, store.view(torch.int64).flatten()[:10].view(2, 5), out=(store, None))
    grad = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        rotary(grad, k, p)
    with torch.no_grad():
        rotary(grad, k, p)
    a, b = rotary(q[:0], k[:0], p[:, :0])
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)
    a, b = rotary(q[:, :0], k, p)
    assert a.shape == (5, 0, 64) and torch.equal(b, k)


# --------------------------------------------------------------------------- moved tokens

@pytest.mark.parametrize("dim,heads,page", [(64, 3, 16), (128, 8, 64), (256, 1, 32)])
@pytest.mark.parametrize("tokens", [1, 2, 511, 513, 1024, 1025, 3000])
def test_move(dim, heads, page, tokens):
    """Chains, cycles and copies: every target holds what its source held before the call; the rest is untouched."""
    pages = -(-2 * tokens // page) + 2
    cache = _random_cache(pages, page, heads, dim, tokens)
    arrays = (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)
    g = torch.Generator().manual_seed(tokens)
    for kind in ("apart", "permuted", "shifted", "one source"):
        before = [t.clone() for t in arrays]
        slots = torch.randperm(pages * page, generator=g).cuda()
        source, target = {"apart": (slots[:tokens], slots[tokens:2 * tokens]), "permuted": (slots[:tokens], slots[:tokens].flip(0)),
                          "shifted": (slots[1:tokens + 1], slots[:tokens]),
                          "one source": (slots[:1].expand(tokens), slots[:tokens])}[kind]
        cache.move(source, target)
        for t, old in zip(arrays, before):
            want = old.clone()
            want[target // page, :, target % page] = old[source // page, :, source % page]
            assert torch.equal(t, want)


@pytest.mark.parametrize("tokens", [6, 2000])
def test_move_skips_slots_outside_the_cache(tokens):
    cache = _random_cache(200, 16, 2, 64, 1)
    before = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    source, target = torch.arange(tokens, device="cuda"), torch.arange(tokens, device="cuda")
    source[0::2] = torch.tensor([-1, 3200, 1 << 40], device="cuda").repeat(tokens)[: len(source[0::2])]
    target[1::2] = torch.tensor([-5, 3201, -(1 << 62)], device="cuda").repeat(tokens)[: len(target[1::2])]
    cache.move(source, target)
    for t, old in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), before):
        assert torch.equal(t, old)
    cache.move(source[:0], target[:0])
    for args, text in (((source[:3], target), "same number"), ((source.int(), target), "dtype"), ((source.cpu(), target), "must be on"),
                       ((source.view(2, -1), target), "dimensions")):
        with pytest.raises(ValueError, match=text):
            cache.move(*args)


# --------------------------------------------------------------------------- together

def test_attend_refuses_bad_masks():
    cache = m.Int4KVCache(4, 16, 2, 64)
    q, table, length, starts = _normal((3, 4, 64), 2, torch.float16), _int32([[0, 1], [2, 3]]), _int32([9, 8]), _int32([0, 2, 3])
    bits = torch.zeros((3, 1), dtype=torch.int64, device="cuda")
    for kw, text in ((dict(sinks=-1, window=4), "sinks must not"), (dict(sinks=2), "sinks need a window"),
                     (dict(ancestors=bits.int()), "dtype"), (dict(ancestors=bits[:2]), "shape"), (dict(ancestors=bits[:, 0]), "dimensions"),
                     (dict(ancestors=bits[:, :0]), "shape"), (dict(ancestors=bits, causal=False), "ancestors need"),
                     (dict(ancestors=bits.cpu()), "must be on"),
                     (dict(ancestors=bits.expand(3, 1), out=torch.zeros((3, 4, 64), device="cuda")), "dtype")):
        with pytest.raises(ValueError, match=text):
            cache.attend(q, table, length, query_offsets=starts, max_query_tokens=2, **kw)
    with pytest.raises(ValueError, match="ancestors need"):
        cache.attend(q[:2], table, length, ancestors=bits[:2])
    with pytest.raises(TypeError, match="tensor"):
        cache.attend(q, table, length, query_offsets=starts, max_query_tokens=2, ancestors=[1, 2, 3])
    store = torch.zeros(3 * 4 * 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        cache.attend(q, table, length, query_offsets=starts, max_query_tokens=2, out=store.view(3, 4, 64),
                     ancestors=store[:12].view(torch.int64).view(3, 1))


def _step(cache, pages, rotary, qkv, tokens, rows, heads, kv, most, base=None, parents=None, window=None, sinks=0):
    """A step: pages, rotary positions, append, attention.  Returns its output, the rows' slots and what went in."""
    offsets, slots, positions = pages.extend(tokens, rows)
    ancestors = None
    if parents is not None:  # a node's position is its depth past the context
        ancestors, depths = m.draft_ancestors(parents, offsets, max_query_tokens=most)
        sequence = torch.bucketize(torch.arange(rows, device="cuda"), offsets[1:].long(), right=True)
        positions = base[sequence] + depths
    query, keys = rotary(qkv[:, :heads], qkv[:, heads:heads + kv], positions)
    cache.append(keys, qkv[:, heads + kv:], slots)
    out = cache.attend(query, pages.page_table, pages.lengths, query_offsets=offsets, max_query_tokens=most, window=window,
                       sinks=sinks, ancestors=ancestors)
    return out, slots, query


@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 5)])
def test_a_tree_is_checked_and_its_path_kept(window, sinks):
    """Prompts, a tree of drafts, its accepted path moved into place, the rest taken back, a token after it: bit for bit
    what the cache holds when the path is appended without the tree; and attention agrees row by row."""
    heads, kv, dim, page, b = 8, 2, 64, 16, 3
    rotary = m.Rotary(dim)
    prompt, tree = [70, 5, 33], [_tree(20, 1), _tree(7, 2), _tree(12, 3)]
    sizes = [len(t) for t in tree]
    g = torch.Generator(device="cuda").manual_seed(5)

    def made(n):
        return torch.randn((n, heads + 2 * kv, dim), generator=g, device="cuda").to(torch.bfloat16)

    def fresh():
        return m.Int4KVCache(40, page, kv, dim), m.PageTable(40, page, b, 12)

    first, draft, after = made(sum(prompt)), made(sum(sizes)), made(b)
    cache, pages = fresh()
    _step(cache, pages, rotary, first, _int32(prompt), sum(prompt), heads, kv, max(prompt), window=window, sinks=sinks)
    base = pages.lengths.clone()
    out, slots, _ = _step(cache, pages, rotary, draft, _int32(sizes), sum(sizes), heads, kv, max(sizes), base=base,
                          parents=_int32([p for t in tree for p in t]), window=window, sinks=sinks)
    # The path to each tree's last node is accepted.
    starts, paths = [0] + np.cumsum(sizes).tolist(), []
    for t in tree:
        path, at = [], len(t) - 1
        while at >= 0:
            path.append(at)
            at = t[at]
        paths.append(path[::-1])
    rows = torch.tensor([starts[s] + i for s, path in enumerate(paths) for i in path], device="cuda")
    places = torch.tensor([starts[s] + i for s, path in enumerate(paths) for i in range(len(path))], device="cuda")
    cache.move(slots[rows], slots[places])
    pages.truncate(base + _int32([len(p) for p in paths]))
    last, _, _ = _step(cache, pages, rotary, after, _int32([1] * b), b, heads, kv, 1, window=window, sinks=sinks)

    other, table = fresh()
    _step(other, table, rotary, first, _int32(prompt), sum(prompt), heads, kv, max(prompt), window=window, sinks=sinks)
    want, _, _ = _step(other, table, rotary, draft[rows], _int32([len(p) for p in paths]), len(rows), heads, kv,
                       max(len(p) for p in paths), window=window, sinks=sinks)
    want_last, _, _ = _step(other, table, rotary, after, _int32([1] * b), b, heads, kv, 1, window=window, sinks=sinks)
    assert pages.lengths.tolist() == table.lengths.tolist() == [n + len(p) + 1 for n, p in zip(prompt, paths)]
    for s, n in enumerate(pages.lengths.tolist()):
        j = torch.arange(n, device="cuda")
        one = cache.read(cache.slots(pages.page_table, torch.full_like(j, s), j), dtype=torch.float32)
        two = other.read(other.slots(table.page_table, torch.full_like(j, s), j), dtype=torch.float32)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    # The same numbers in another order of sums: each off by half a step of bf16 and 2^-10 of values up to about 4.
    assert ((out[rows].double() - want.double()).abs() <= 2.0**-7 * want.double().abs() + 2.0**-9 * 4).all()
    assert ((last.double() - want_last.double()).abs() <= 2.0**-7 * want_last.double().abs() + 2.0**-9 * 4).all()


@pytest.mark.parametrize("tokens", [200, 3000])
def test_kernels_that_start_early_wait_for_what_they_read(tokens):
    """A chain of calls whose inputs the kernel just before makes (torch's or this library's), run on and on, gives what it
    gives with a wait after every call."""
    heads, dim, page, b = 4, 64, 16, 5
    pages = -(-tokens // page) + b

    def run(wait):
        g = torch.Generator(device="cuda").manual_seed(tokens)
        cache, table, rotary = m.Int4KVCache(2 * pages, page, heads, dim), m.PageTable(2 * pages, page, b, 2 * pages), m.Rotary(dim)
        share = _int32([tokens // b] * b)
        most, results = tokens // b, []
        x = torch.randn((tokens, heads, dim), generator=g, device="cuda").to(torch.bfloat16)
        parents = torch.arange(-1, most - 1, dtype=torch.int32, device="cuda").repeat(b) if most <= 1024 else None
        for step in range(6):
            offsets, slots, positions = table.extend(share, tokens)
            wait()
            q, k = rotary(x, x, positions)
            wait()
            cache.append(k, q, slots)
            wait()
            order = torch.randperm(tokens, generator=g, device="cuda")
            wait()
            cache.move(slots[order] * 1, slots.flip(0) + 0)  # the slots come from the kernels just before
            wait()
            bits, depths = m.draft_ancestors(parents * 1, offsets, max_query_tokens=most)
            wait()
            a = cache.attend(q, table.page_table, table.lengths, query_offsets=offsets, max_query_tokens=most, ancestors=bits)
            wait()
            w = cache.attend(a, table.page_table, table.lengths, query_offsets=offsets, max_query_tokens=most, window=20, sinks=3)
            wait()
            x = (a + w).clamp(-3, 3)
            table.truncate(table.lengths - (share - 1 - step))
            wait()
            results.append((x, depths, positions, table.lengths.clone()))
        torch.cuda.synchronize()
        return [t.clone() for r in results for t in r] + [cache.k_codes, cache.v_scales, table.page_table, table.free_pages]

    want = run(torch.cuda.synchronize)
    for _ in range(3):
        for got, w in zip(run(lambda: None), want):
            assert torch.equal(got, w)


def test_graphs_and_streams():
    """The step captured into two graphs that live at once, replayed in turn and with new inputs in place; and calls on
    two streams at once."""
    heads, kv, dim, b = 8, 2, 128, 5
    rotary = m.Rotary(dim, sections=[20, 22, 22])
    cache, pages = m.Int4KVCache(300, 16, kv, dim), m.PageTable(300, 16, b, 60)
    lengths = [600, 3, 100, 0, 257]
    _, slots, _ = pages.extend(_int32(lengths), sum(lengths))
    kvs = _normal((sum(lengths), 2 * kv, dim), 1, torch.bfloat16)
    cache.append(kvs[:, :kv], kvs[:, kv:], slots)
    before = pages.lengths.clone()
    qkv = _normal((4 * b, heads + 2 * kv, dim), 2, torch.bfloat16)
    tokens, positions = _int32([4] * b), torch.randint(0, 999, (3, 4 * b), device="cuda")
    parents = _int32([-1, 0, 0, 1] * b)

    def step():
        offsets, slots, _ = pages.extend(tokens, 4 * b)
        bits, depths = m.draft_ancestors(parents, offsets, max_query_tokens=4)
        query, keys = rotary(qkv[:, :heads], qkv[:, heads:heads + kv], positions)
        cache.append(keys, qkv[:, heads + kv:], slots)
        a = cache.attend(query, pages.page_table, pages.lengths, query_offsets=offsets, max_query_tokens=4, ancestors=bits)
        w = cache.attend(query, pages.page_table, pages.lengths, query_offsets=offsets, max_query_tokens=4, window=64, sinks=8)
        cache.move(slots.flip(0), slots)
        pages.truncate(before)
        return a, w

    want = [t.clone() for t in step()]
    again = step()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for i in (0, 1, 0):
        graphs[i].replay()
        assert all(torch.equal(a, b) for a, b in zip(want, outs[i]))
    qkv.copy_(_normal((4 * b, heads + 2 * kv, dim), 3, torch.bfloat16))
    positions.add_(17)
    parents.copy_(_int32([-1, -1, 1, 1] * b))
    fresh = [t.clone() for t in step()]
    for i in (1, 0):
        graphs[i].replay()
        assert all(torch.equal(a, b) for a, b in zip(fresh, outs[i]))
    # Calls that only read, on two streams at once.
    offsets, _, _ = pages.extend(tokens, 4 * b)
    bits, _ = m.draft_ancestors(parents, offsets, max_query_tokens=4)
    query = qkv[:, :heads]

    def reads():
        return (cache.attend(query, pages.page_table, pages.lengths, query_offsets=offsets, max_query_tokens=4, ancestors=bits),
                cache.attend(query, pages.page_table, pages.lengths, query_offsets=offsets, max_query_tokens=4, window=64, sinks=8),
                rotary(query, None, positions)[0])

    alone = reads()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results += [reads() for _ in range(5)]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in results for a, b in zip(r, alone))


@pytest.mark.parametrize("window,sinks", [(None, 0), (24, 3)])
def test_example_answers_with_drafts(window, sinks):
    """The example runs, keeps one to three tokens a step, and what it keeps is a path of what it drafted."""
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import answer_with_drafts

    answer, counts = answer_with_drafts.main(prompts=(20, 1, 33), tokens=6, window=window, sinks=sinks)
    assert answer.shape == (3, 6, 3) and counts.shape == (3, 6)
    assert ((counts >= 1) & (counts <= 3)).all()
    assert torch.equal((answer >= 0).sum(dim=2), counts) and ((answer[..., 0] >= 0) & (answer[..., 0] < 1000)).all()
