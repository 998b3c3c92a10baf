"""The serving step's operators where their ranges end: prompts under a window from their first token on, blocks of many small
segments, masks wider than any tree, arrays between guard words, steps that nothing waits for."""

import pytest

import maxsim_b200 as m
from maxsim_b200 import _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_kv4 import DTYPES, _normal, _random_cache, _tables  # noqa: E402
from test_gpu_reader_step import _check_rows, _int32, engine  # noqa: E402, F401


# --------------------------------------------------------------------------- prompts under a window with sinks

def _window_mask(length, rows, window, sinks):
    """[rows, length]: the last `rows` tokens, each up to its own, the last `window` of these and the first `sinks`."""
    p, j = torch.arange(length - rows, length).unsqueeze(1), torch.arange(length)
    return (j <= p) & ((j > p - window) | (j < sinks))


def _check_prompts(dim, heads, shared, page, dtype, lengths, rows, window, sinks, seed=0):
    pages = sum(-(-n // page) for n in lengths) + 2
    cache, table = _random_cache(pages, page, heads, dim, seed), _tables(lengths, page, pages, seed=seed)
    offsets = [sum(rows[:b]) for b in range(len(rows) + 1)]
    query = _normal((offsets[-1], heads * shared, dim), seed + 9, DTYPES[dtype], 1.5)
    got, lse = cache.attend(query, table, _int32(lengths), query_offsets=_int32(offsets), max_query_tokens=max(rows),
                            window=window, sinks=sinks, return_lse=True)
    masks = [_window_mask(n, r, window, sinks) for n, r in zip(lengths, rows)]
    _check_rows(got, lse, query, cache, table, lengths, offsets, masks, dim**-0.5)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [24, 256, 1024])
@pytest.mark.parametrize("sinks", [4, 64, 300])
def test_sinks_of_prompts_from_their_first_token(engine, dim, window, sinks):  # noqa: F811
    """Rows whose window has left the sinks beside rows whose window is still over them, in one sequence."""
    _check_prompts(dim, 2, 4, 16, "bf16", [200, 512, 700, 1536], [200, 512, 700, 512], window, sinks, seed=sinks)


@pytest.mark.parametrize("dim,heads,shared,length,rows,window,sinks", [
    (128, 8, 1, 200, 200, 24, 4), (128, 2, 4, 512, 512, 256, 4), (256, 1, 1, 300, 300, 1, 1), (256, 8, 4, 1536, 512, 1024, 4),
    (64, 1, 4, 2500, 2500, 130, 33), (128, 1, 2, 2500, 1000, 700, 1000), (128, 1, 1, 5000, 5000, 16, 97)])
def test_sinks_of_one_prompt(dim, heads, shared, length, rows, window, sinks):
    """One sequence, by the kernel that the sizes choose: a cluster a segment, or ranges that end among the sinks, between
    them and the window, within it."""
    _check_prompts(dim, heads, shared, 32, "f16", [length], [rows], window, sinks, seed=length)


@pytest.mark.parametrize("window,sinks", [(24, 4), (256, 64)])
def test_the_example_sees_a_long_prompts_sinks(monkeypatch, window, sinks):
    """Every layer's attention to prompts of 300 tokens and fewer, in 64 bits."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import answer_with_drafts

    plain, prompts, seen = m.Int4KVCache.attend, (300, 5, 80), []

    def attend(cache, query, page_table, lengths, **kw):
        out = plain(cache, query, page_table, lengths, **kw)
        if kw.get("ancestors") is None:
            got, lse = plain(cache, query, page_table, lengths, return_lse=True, **kw)
            assert torch.equal(got, out)
            offsets = kw["query_offsets"].tolist()
            masks = [_window_mask(n, n, window, sinks) for n in prompts]
            _check_rows(got, lse, query, cache, page_table, lengths.tolist(), offsets, masks, query.shape[2]**-0.5)
            seen.append(offsets)
        return out

    monkeypatch.setattr(m.Int4KVCache, "attend", attend)
    answer_with_drafts.main(prompts=prompts, tokens=1, window=window, sinks=sinks)
    assert seen == [[0, 300, 305, 385]] * 2


# --------------------------------------------------------------------------- kernels that start early

@pytest.mark.parametrize("dim,most", [(64, 3), (128, 12), (128, 70), (256, 12)])
def test_inputs_that_the_kernel_before_writes_anew(engine, dim, most):  # noqa: F811
    """Page table entries, masks, queries and codes at the same addresses step after step, each written by the kernel just
    before the one that reads it, while that one is already there."""
    b, heads, kv, page = 9, 8, 2, 16
    rows, parents = b * most, _int32([-1] + [i // 2 for i in range(most - 1)]).repeat(b)
    tokens, flat = _int32([most] * b), _int32([-1, *range(most - 1)]).repeat(b)
    x = _normal((20, rows, heads + 2 * kv, dim), dim + most, torch.bfloat16)

    def run(wait):
        cache, table, rotary = m.Int4KVCache(400, page, kv, dim), m.PageTable(400, page, b, 40), m.Rotary(dim)
        query, kept, results = torch.empty((rows, heads, dim), dtype=torch.bfloat16, device="cuda"), torch.empty(0), []
        before = _int32([5 * i for i in range(b)])
        _, slots, _ = table.extend(before, 180)
        cache.append(x[0, :1, :kv].expand(180, kv, dim), x[0, :1, kv:2 * kv].expand(180, kv, dim), slots)
        for step in range(20):
            now = x[step]
            offsets, slots, positions = table.extend(tokens, rows)
            wait()
            cache.append(now[:, heads:heads + kv], now[:, heads + kv:], slots)
            wait()
            cache.move(slots.flip(0), slots)
            wait()
            bits, depths = m.draft_ancestors(parents if step % 2 else flat, offsets, max_query_tokens=most)
            wait()
            rotary(now[:, :heads], None, positions, out=(query, None))
            wait()
            a = cache.attend(query, table.page_table, table.lengths, query_offsets=offsets, max_query_tokens=most, ancestors=bits)
            wait()
            rotary(now[:, :heads], None, depths, out=(query, None))
            wait()
            w = cache.attend(query, table.page_table, table.lengths, query_offsets=offsets, max_query_tokens=most, window=9, sinks=4)
            wait()
            kept = table.lengths - (tokens - step % 2)  # every second step keeps a token
            table.truncate(kept)
            wait()
            if step % 5 == 4:  # other pages for all
                table.truncate(torch.zeros_like(tokens))
                wait()
                table.extend(kept.flip(0), 400)
                wait()
            results += [a, w, table.lengths.clone(), table.page_table.clone()]
        torch.cuda.synchronize()
        return results

    want = run(torch.cuda.synchronize)
    assert not any(torch.isnan(t).any() for t in want)
    for _ in range(3):
        for got, w in zip(run(lambda: None), want):
            assert torch.equal(got, w)


@pytest.mark.parametrize("dim,shared,batch", [(64, 8, 400), (128, 4, 150), (128, 64, 90)])
@pytest.mark.parametrize("tree", [False, True])
def test_segments_of_one_and_two_row_tiles_in_turn(dim, shared, batch, tree):
    """Dozens of segments for each block of the kernel for many rows, of few tiles of tokens: runs of segments with one
    tile of rows, where half of the kernel's warps have no products and only keep up, with some of two, of more than 256
    rows and without tokens among them."""
    sizes = [1, 2, 3, 1, 1, 128 // shared, 1, 2, 0, 1, 128 // shared + 1, 1, 1, 256 // shared + 1, 1, 2, 256 // shared, 1, 1, 0]
    rows = [sizes[(7 * b) % 20 if b % 60 < 30 else b % 5] for b in range(batch)]
    lengths = [max(0, n + [0, 40, 3, 130, 0, 300, 17][b % 7] - (n if b % 23 == 5 else 0)) for b, n in enumerate(rows)]
    trees = [[(i - 1) // 2 for i in range(n)] for n in rows]
    pages = sum(-(-n // 16) for n in lengths) + 2
    cache, table = _random_cache(pages, 16, 2, dim, 3), _tables(lengths, 16, pages, seed=4)
    offsets = [sum(rows[:b]) for b in range(batch + 1)]
    query = _normal((offsets[-1], 2 * shared, dim), 5, torch.float16, 1.5)
    kw = dict(query_offsets=_int32(offsets), max_query_tokens=max(rows), return_lse=True)
    if tree:
        kw["ancestors"], _ = m.draft_ancestors(_int32([p for t in trees for p in t]), kw["query_offsets"], max_query_tokens=max(rows))
        masks = [_tree_mask(n, t) for n, t in zip(lengths, trees)]
    else:
        kw.update(window=50, sinks=7)
        masks = [_window_mask(n, r, 50, 7) for n, r in zip(lengths, rows)]
    _lib.set_option("kv4_engine", 2)
    try:
        results = [cache.attend(query, table, _int32(lengths), **kw) for _ in range(4)]
    finally:
        _lib.set_option("kv4_engine", 0)
    for got, lse in results[1:]:
        assert torch.equal(got, results[0][0]) and torch.equal(lse, results[0][1])
    _check_rows(*results[0], query, cache, table, lengths, offsets, masks, dim**-0.5)


def _tree_mask(length, parents):
    """[nodes, length]: all before the nodes, and each node's path."""
    rows, first = len(parents), length - len(parents)
    mask = torch.zeros((rows, length), dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            mask[i] = mask[p]
        elif first > 0:
            mask[i, :first] = True
        if first + i >= 0:
            mask[i, first + i] = True
    return mask


# --------------------------------------------------------------------------- masks of drafted trees, from C

def _draft_ancestors(parents, offsets, most, words, ancestors, depths):
    rows, batch = ancestors.shape[0], offsets.shape[0] - 1
    _lib.check(_lib.lib.msb_draft_ancestors_device(parents.data_ptr(), rows, offsets.data_ptr(), batch, most, words,
                                                   ancestors.data_ptr(), depths.data_ptr(), 0,
                                                   torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("rows,words", [(5, 1), (70, 2), (70, 3), (70, 16), (70, 17), (70, 100), (1024, 2**21)])
def test_masks_wider_than_their_trees(rows, words):
    """Words past a tree's nodes are 0, however wide the caller's rows are: the last case has 2^31 words, 17 GB."""
    if 8 * rows * words > torch.cuda.mem_get_info()[0] // 2:
        pytest.skip("not enough memory")
    ancestors = torch.full((rows + 1, words), -1, dtype=torch.int64, device="cuda")
    depths = torch.full((rows + 1,), -1, dtype=torch.int32, device="cuda")
    parents = torch.tensor([i - 1 if i % 50 else i - 3 for i in range(rows + 1)], dtype=torch.int32, device="cuda")
    _draft_ancestors(parents, _int32([0, rows]), rows, words, ancestors, depths)
    want, want_depths = m.draft_ancestors(parents[:rows], _int32([0, rows]), max_query_tokens=rows)
    held = want.shape[1]
    assert torch.equal(ancestors[:rows, :held], want) and torch.equal(depths[:rows], want_depths)
    assert not ancestors[:, held:].any() and not ancestors[rows].any() and depths[rows] == 0


def test_rows_of_no_sequence_at_all():
    """Without sequences every row's mask and depth is 0, from C as from Python; nothing past the rows is written."""
    ancestors = torch.full((6, 3), -1, dtype=torch.int64, device="cuda")
    depths = torch.full((6,), -1, dtype=torch.int32, device="cuda")
    parents, offsets = _int32([-1, 0, 1, 2, 3]), _int32([0])
    _draft_ancestors(parents, offsets, 5, 3, ancestors[:5], depths[:5])
    assert not ancestors[:5].any() and not depths[:5].any() and (ancestors[5] == -1).all() and depths[5] == -1
    for _ in range(3):  # fresh memory that holds something
        torch.full((1000,), -1, dtype=torch.int64, device="cuda")
        bits, depths = m.draft_ancestors(parents, offsets)
        assert bits.shape == (5, 1) and not bits.any() and not depths.any()


def test_the_examples_steps_wait_for_nothing(monkeypatch):
    """The host asks for step after step without waiting for the GPU: no copy from pageable memory and no read-back from the
    first step's table call on."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import answer_with_drafts

    extend, calls = m.PageTable.extend, []

    def watched(table, tokens, rows):
        if calls:  # the first call is the prompts'
            torch.cuda.set_sync_debug_mode("error")
        calls.append(rows)
        return extend(table, tokens, rows)

    monkeypatch.setattr(m.PageTable, "extend", watched)
    try:
        answer, counts = answer_with_drafts.main(prompts=(20, 1, 33), tokens=5, window=24, sinks=3)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert calls == [54] + [15] * 5
    assert torch.equal((answer >= 0).sum(dim=2), counts) and ((counts >= 1) & (counts <= 3)).all()


# --------------------------------------------------------------------------- page tables

@pytest.mark.parametrize("sequences", [1, 3, 256, 257, 1500])
@pytest.mark.parametrize("lengths,count,page", [(1 << 30, 1 << 30, -5), (-9, -9, 1 << 30), (63, 6, -(1 << 31)), (64, 0, 7),
                                                (0, 6, 7), (17, 1 << 30, 1 << 30), (40, 3, 3)])
def test_page_tables_that_hold_nonsense_keep_to_their_arrays(sequences, lengths, count, page):
    """Whatever lengths, counts and ids the four arrays hold, nothing beside any of them is written, and what is read of them
    is theirs: all four lie between guard words, whose values as lengths, counts or ids would show in the results."""
    guard, gap = 123456789, 512
    sizes = (4 * sequences, sequences, 6, 1)  # table [sequences, 4], lengths, stack of 6, its count
    results = []
    for value in (guard, -guard):
        store = torch.full((sum(sizes) + gap * 5,), value, dtype=torch.int32, device="cuda")
        parts, inside, at = [], torch.zeros_like(store, dtype=torch.bool), gap
        for n, fill in zip(sizes, (page, lengths, page, count)):
            parts.append(store[at:at + n])
            parts[-1].fill_(fill)
            inside[at:at + n] = True
            at += n + gap
        table = m.PageTable.from_tensors(parts[0].view(sequences, 4), *parts[1:], page_size=16)
        tokens = torch.full((sequences,), 7, dtype=torch.int32, device="cuda")
        seen = []
        for call in ("extend", "truncate", "extend"):
            if call == "extend":
                seen += table.extend(tokens, 7 * sequences)
                assert ((seen[-1] >= -1) & (seen[-1] < 64)).all()
            else:
                table.truncate(torch.full((sequences,), -3, dtype=torch.int32, device="cuda"))
                assert (table.lengths == 0).all() and 0 <= table.free_count.item() <= 6
            assert (store[~inside] == value).all()
            seen += [t.clone() for t in parts]
        results.append(seen)
    assert all(torch.equal(a, b) for a, b in zip(*results))
