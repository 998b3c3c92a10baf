"""The 4-bit key/value cache: written, read back and attended over, against plain arithmetic in 64 bits."""

import numpy as np
import pytest

import maxsim_b200 as m

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _normal(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _values(codes, scales):
    """64-bit values of code bytes [..., d / 2] and scales [...]."""
    c = codes.to(torch.int16)
    out = torch.stack((((c & 15) ^ 8) - 8, ((c >> 4) ^ 8) - 8), dim=-1).flatten(-2).double()
    return out * scales.double().unsqueeze(-1)


def _random_cache(pages, page, heads, dim, seed):
    """A cache whose every slot holds something, keys a little wider than values."""
    cache = m.Int4KVCache(pages, page, heads, dim)
    slots = torch.arange(pages * page, device="cuda")
    cache.append(_normal((pages * page, heads, dim), seed), _normal((pages * page, heads, dim), seed + 1, scale=0.3), slots)
    return cache


def _packed(x):
    """Code bytes and scales of fp32 vectors [n, d]: scale fl(max|x| * fl(1/7)), 0 -> 1; codes rint(fl(x / scale))."""
    x = x.float().cpu().numpy().reshape(-1, x.shape[-1])
    scale = np.abs(x).max(axis=1) * np.float32(1.0 / 7.0)
    scale[scale == 0] = 1
    codes = np.clip(np.rint(x / scale[:, None]), -7, 7).astype(np.int8)
    return ((codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)).astype(np.uint8), scale, codes


# --------------------------------------------------------------------------- write and read

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,page,tokens", [(64, 1, 16, 1), (64, 3, 32, 77), (128, 8, 16, 64), (128, 2, 64, 1001),
                                                   (256, 5, 128, 130), (128, 1, 1024, 2050)])
def test_append_writes_codes_and_scales(dtype, dim, heads, page, tokens):
    """Codes and scales byte for byte, within two units in the last place of the corpus packer's scale; other slots
    stay as they were."""
    pages = -(-tokens // page) + 1
    cache = m.Int4KVCache(pages, page, heads, dim)
    before = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    g = torch.Generator().manual_seed(tokens)
    slots = torch.randperm(pages * page, generator=g)[:tokens].cuda()
    keys, values = _normal((tokens, heads, dim), 1, DTYPES[dtype]), _normal((tokens, heads, dim), 2, DTYPES[dtype], 40.0)
    cache.append(keys, values, slots)
    untouched = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    untouched[slots] = False
    for x, codes, scales, old_codes, old_scales in ((keys, cache.k_codes, cache.k_scales, before[0], before[1]),
                                                    (values, cache.v_codes, cache.v_scales, before[2], before[3])):
        want_codes, want_scales, _ = _packed(x)
        corpus = m.pack_int4_symmetric(x.float().cpu().numpy().reshape(-1, dim), scale_granularity="token")
        np.testing.assert_allclose(want_scales, corpus.token_scale, rtol=2.0**-22)
        by_slot = codes.transpose(1, 2).reshape(pages * page, heads, dim // 2)
        scale_by_slot = scales.transpose(1, 2).reshape(pages * page, heads)
        np.testing.assert_array_equal(by_slot[slots].cpu().numpy().reshape(-1, dim // 2), want_codes)
        np.testing.assert_array_equal(scale_by_slot[slots].cpu().numpy().reshape(-1), want_scales)
        old = old_codes.transpose(1, 2).reshape(pages * page, heads, dim // 2)
        assert torch.equal(by_slot[untouched], old[untouched])
        assert torch.equal(scale_by_slot[untouched], old_scales.transpose(1, 2).reshape(pages * page, heads)[untouched])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,page", [(64, 3, 16), (128, 8, 64), (256, 1, 32)])
def test_read_rounds_once(dtype, dim, heads, page):
    cache = _random_cache(5, page, heads, dim, seed=7)
    slots = torch.randperm(5 * page, generator=torch.Generator().manual_seed(3))[: 4 * page + 1].cuda()
    keys, values = cache.read(slots, dtype=DTYPES[dtype])
    for got, codes, scales in ((keys, cache.k_codes, cache.k_scales), (values, cache.v_codes, cache.v_scales)):
        want = _values(codes, scales)[slots // page, :, slots % page]
        assert got.dtype == DTYPES[dtype] and got.shape == want.shape
        # code * scale is rounded to fp32 and, for 16-bit outputs, that to the output's type
        assert torch.equal(got, want.float().to(DTYPES[dtype]))


def test_ties_zeros_small_and_large_vectors():
    """Quotients at .5 round to even; zero vectors get scale 1; the smallest and largest fp32 values."""
    x = torch.zeros((6, 1, 64), device="cuda")
    x[1, 0, :8] = torch.tensor([7.0, 3.5, 2.5, 1.5, 0.5, -0.5, -3.5, -2.5])
    x[2, 0, 5] = -1e-45  # max / 7 is 0: scale 1
    x[3, 0, :2] = torch.tensor([1e-38, -4e-39])
    x[4, 0, :2] = torch.tensor([3.4e38, -1.7e38])
    x[5, 0, 63] = -0.0
    cache = m.Int4KVCache(1, 16, 1, 64)
    cache.append(x, -x, torch.arange(6, device="cuda"))
    codes, scales, _ = _packed(x)
    np.testing.assert_array_equal(cache.k_codes[0, 0, :6].cpu().numpy(), codes)
    np.testing.assert_array_equal(cache.k_scales[0, 0, :6].cpu().numpy(), scales)
    np.testing.assert_array_equal(cache.v_scales[0, 0, :6].cpu().numpy(), scales)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_vectors_that_are_not_finite(bad, dtype):
    """One vector with such a value reads back as NaN; its neighbours are what they were."""
    x = _normal((4, 2, 128), 5, DTYPES[dtype])
    y = x.clone()
    y[2, 1, 77] = bad
    cache, clean = m.Int4KVCache(1, 16, 2, 128), m.Int4KVCache(1, 16, 2, 128)
    slots = torch.arange(4, device="cuda")
    cache.append(x, y, slots)
    clean.append(x, x, slots)
    got, want = cache.read(slots, dtype=torch.float32), clean.read(slots, dtype=torch.float32)
    assert torch.equal(got[0], want[0])
    assert torch.isnan(got[1][2, 1]).all()
    keep = torch.ones((4, 2), dtype=torch.bool, device="cuda")
    keep[2, 1] = False
    assert torch.equal(got[1][keep], want[1][keep])
    assert not cache.v_codes[0, 1, 2].any()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strided_and_unaligned_inputs(dim, dtype):
    """Keys and values as views: heads before tokens, a slice of a fused projection, odd offsets, broadcast heads."""
    t, h = 37, 3
    fused = _normal((t, 3 * h * dim + 5), 11, DTYPES[dtype])
    layouts = [
        fused[:, 1 : 1 + h * dim].unflatten(1, (h, dim)),  # rows start off any 4-byte boundary
        fused[:, h * dim : 2 * h * dim].unflatten(1, (h, dim)),
        _normal((h, t, dim), 12, DTYPES[dtype]).transpose(0, 1),
        _normal((t, 1, dim), 13, DTYPES[dtype]).expand(t, h, dim),
        _normal((t, h, 2 * dim), 14, DTYPES[dtype])[:, :, ::2],
    ]
    slots = torch.randperm(64, generator=torch.Generator().manual_seed(1))[:t].cuda()
    for x in layouts:
        one, two = m.Int4KVCache(4, 16, h, dim), m.Int4KVCache(4, 16, h, dim)
        one.append(x, x.contiguous(), slots)
        two.append(x.contiguous(), x, slots)
        assert torch.equal(one.k_codes, two.k_codes) and torch.equal(one.k_scales, two.k_scales)
        assert torch.equal(one.v_codes, one.k_codes) and torch.equal(two.v_codes, two.k_codes)
        assert torch.equal(one.v_scales, two.k_scales)


def test_slots_outside_the_cache():
    cache = _random_cache(2, 16, 2, 64, seed=3)
    before = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    x = _normal((5, 2, 64), 1)
    slots = torch.tensor([-1, 32, 1 << 40, -(1 << 62), 33], device="cuda")
    cache.append(x, x, slots)
    for t, old in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), before):
        assert torch.equal(t, old)
    keys, values = cache.read(torch.tensor([-1, 3, 32, 1 << 40], device="cuda"), dtype=torch.float32)
    assert not keys[[0, 2, 3]].any() and not values[[0, 2, 3]].any() and keys[1].any()
    cache.append(x[:0], x[:0], slots[:0])
    assert cache.read(slots[:0])[0].shape == (0, 2, 64)


# --------------------------------------------------------------------------- attention

def _plain(query, cache, table, lengths, offsets, scale, causal=True, window=None):
    """64-bit attention, lse, and per row the derived error bound (see _check)."""
    rows, heads, dim = query.shape
    shared = heads // cache.num_kv_heads
    page = cache.page_size
    out = torch.zeros((rows, heads, dim), dtype=torch.float64, device="cuda")
    lse = torch.full((rows, heads), -torch.inf, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    slack = torch.zeros_like(lse)
    for b, length in enumerate(lengths):
        lo, hi = offsets[b], offsets[b + 1]
        if length == 0 or hi == lo:
            continue
        j = torch.arange(length, device="cuda")
        pages = table[b].long()[j // page]
        held = (pages >= 0) & (pages < cache.num_pages)
        pages = torch.where(held, pages, 0)
        for h in range(cache.num_kv_heads):
            k = _values(cache.k_codes[pages, h, j % page], cache.k_scales[pages, h, j % page])
            v = _values(cache.v_codes[pages, h, j % page], cache.v_scales[pages, h, j % page])
            q = query[lo:hi, h * shared : (h + 1) * shared].double()
            s = torch.einsum("nsd,jd->nsj", q, k) * scale
            pos = length - (hi - lo) + torch.arange(hi - lo, device="cuda").view(-1, 1, 1)
            seen = held & (j <= pos) if causal else (held & (j >= 0)).expand(hi - lo, 1, length)
            if window:
                seen = seen & (j > pos - window)
            s = s.masked_fill(~seen, -torch.inf)
            any_seen = seen.any(-1)
            top = torch.logsumexp(s, -1)
            p = torch.where(any_seen.unsqueeze(-1), torch.exp(s - top.unsqueeze(-1)), 0.0)
            v = torch.where(seen.any(0).any(0).unsqueeze(-1), v, 0.0)
            at = slice(lo, hi), slice(h * shared, (h + 1) * shared)
            out[at] = torch.einsum("nsj,jd->nsd", p, v)
            lse[at] = torch.where(any_seen, top, -torch.inf)
            bound[at] = torch.einsum("nsj,jd->nsd", p, v.abs())
            # Products are exact; partial sums of one score stay below 80 sum|q| ks and are rounded (or cut) to
            # 24 bits at most dim / 16 + 16 times; so a score is off by at most this much.
            ks = torch.where(seen.any(0).any(0), cache.k_scales[pages, h, j % page].double(), 0.0).nan_to_num(0.0).max()
            slack[at] = q.abs().sum(-1) * ks * scale * 80 * (dim / 16 + 16) * 2.0**-23
    return out, lse, bound, slack


def _check(got, want, lse=None):
    """|got - o| <= eps |o| + (2^-10 + 2 slack) sum p |v|: the output's rounding, the probabilities' rounding to
    fp16 (relative 2^-11, and fp32 exponentials) and the scores' error, which moves numerator and denominator."""
    out, want_lse, bound, slack = want
    eps = 2.0**-8 if got.dtype == torch.bfloat16 else 2.0**-10
    limit = eps * out.abs() + (2.0**-10 + 2 * slack.unsqueeze(-1)) * bound + 1e-7
    off = (got.double() - out).abs()
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    ok = (off <= limit) | torch.isnan(out)
    assert ok.all(), f"worst {(off / limit).nan_to_num(0).max().item():.3g} of the bound"
    if lse is not None:
        seen = ~torch.isinf(want_lse)
        assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
        assert ((lse.double() - want_lse).abs() <= slack + 1e-5 + 1e-6 * want_lse.abs())[seen & ~torch.isnan(want_lse)].all()


def _tables(lengths, page, pages, extra=1, seed=0):
    """A page table over a random order of pages; entries past a sequence's end name a page outside the cache."""
    per = max(1, -(-max(lengths) // page)) + extra
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    rows = []
    for n in lengths:
        used = -(-n // page)
        rows.append([ids.pop() for _ in range(used)] + [1 << 30] * (per - used))
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def _run(dim, heads, shared, page, dtype, lengths, rows=None, causal=True, window=None, seed=0, scale=None, query=None):
    pages = sum(-(-n // page) for n in lengths) + 2
    cache = _random_cache(pages, page, heads, dim, seed)
    table = _tables(lengths, page, pages, seed=seed)
    offsets = list(range(len(lengths) + 1)) if rows is None else np.concatenate([[0], np.cumsum(rows)]).tolist()
    if query is None:
        query = _normal((offsets[-1], heads * shared, dim), seed + 9, DTYPES[dtype], 1.5)
    got, lse = cache.attend(query, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                            query_offsets=None if rows is None else torch.tensor(offsets, dtype=torch.int32, device="cuda"),
                            max_query_tokens=None if rows is None else max(rows), scale=scale, causal=causal, window=window,
                            return_lse=True)
    want = _plain(query, cache, table, lengths, offsets, dim**-0.5 if scale is None else scale, causal, window)
    _check(got, want, lse)
    return cache, table, query, got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,shared", [(1, 1), (2, 3), (4, 8), (1, 16), (2, 17), (1, 40)])
def test_one_token(dim, heads, shared, dtype):
    """Decode: lengths around every tile edge, an empty sequence, every way of sharing heads."""
    _run(dim, heads, shared, 16, dtype, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 1030])


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
def test_page_sizes(page):
    _run(128, 2, 4, page, "bf16", [page - 1, page, page + 1, 3 * page + 7, 1], seed=page)


@pytest.mark.parametrize("dtype,dim", [("f16", 64), ("bf16", 128), ("f16", 128), ("bf16", 256)])
@pytest.mark.parametrize("shared", [1, 4, 7])
@pytest.mark.parametrize("window", [None, 1, 33, 200])
def test_ragged_rows(dtype, dim, shared, window):
    """Several rows a sequence, causal, some sequences without rows and some with more rows than tokens."""
    _run(dim, 2, shared, 32, dtype, [5, 70, 0, 130, 64, 3, 257], rows=[5, 1, 3, 40, 0, 7, 129], window=window, seed=shared)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,length", [(64, 64), (127, 500), (128, 128), (129, 1000), (300, 1111)])
@pytest.mark.parametrize("shared", [1, 4])
def test_chunks(dim, rows, length, shared):
    _run(dim, 2, shared, 64, "bf16", [length, length // 2 + rows], rows=[rows, rows], seed=rows)


@pytest.mark.parametrize("rows", [None, [3, 1, 20], [200, 1, 64]])
def test_without_causal(rows):
    _run(128, 2, 4, 16, "f16", [100, 33, 250], rows=rows, causal=False)


@pytest.mark.parametrize("window", [1, 5, 64, 1000, 100000])
def test_window_of_one_token(window):
    _run(128, 2, 4, 16, "bf16", [0, 1, 64, 65, 700, 3000], window=window)


@pytest.mark.parametrize("batch,length,heads,shared", [(1, 70001, 2, 4), (2, 40000, 8, 8), (1, 131072, 1, 1), (300, 50, 2, 2)])
def test_long_and_wide(batch, length, heads, shared):
    _run(128, heads, shared, 128, "f16", [length - 37 * b if length > 1000 else length - b % 50 for b in range(batch)], seed=batch)


def test_peaked_scores_and_rising_maxima():
    """Scores that grow along the sequence move the running maximum in every tile."""
    cache = m.Int4KVCache(40, 16, 1, 128)
    direction = _normal((1, 1, 128), 4)
    k = direction * torch.linspace(-3, 3, 640, device="cuda").view(-1, 1, 1) + _normal((640, 1, 128), 5, scale=0.1)
    cache.append(k, _normal((640, 1, 128), 6), torch.arange(640, device="cuda"))
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40)
    for sign in (1, -1):
        q = (sign * direction * 4).expand(1, 4, 128).to(torch.bfloat16)
        got, lse = cache.attend(q, table, torch.tensor([640], dtype=torch.int32, device="cuda"), return_lse=True)
        _check(got, _plain(q, cache, table, [640], [0, 1], 128**-0.5), lse)


@pytest.mark.parametrize("size", [1e-30, 1e-8, 1e8, 1e30])
def test_range_of_bf16(size):
    """Queries and values far outside fp16's range."""
    lengths, page = [100, 40], 16
    cache = m.Int4KVCache(12, page, 2, 128)
    every = torch.arange(12 * page, device="cuda")
    v = _normal((12 * page, 2, 128), 2) * size
    k = _normal((12 * page, 2, 128), 3) / size
    cache.append(k, v, every)
    table = _tables(lengths, page, 12)
    q = (_normal((2, 8, 128), 4) * size).to(torch.bfloat16)
    got = cache.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    out, lse, bound, slack = _plain(q, cache, table, lengths, [0, 1, 2], 128**-0.5)
    _check(got, (out, lse, bound, slack))
    assert ((got.double() - out).abs() <= 2.0**-8 * out.abs() + (2.0**-10 + 2 * slack.unsqueeze(-1)) * bound).all()


def test_values_of_very_different_sizes():
    """Scales of values from 1e-6 to 1e6 in one sequence, and zero vectors among small ones."""
    cache = m.Int4KVCache(8, 16, 1, 64)
    v = _normal((128, 1, 64), 2) * torch.logspace(-6, 6, 128, device="cuda")[torch.randperm(128, generator=torch.Generator().manual_seed(9))].view(-1, 1, 1)
    cache.append(_normal((128, 1, 64), 3), v, torch.arange(128, device="cuda"))
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
    q = _normal((1, 4, 64), 4, torch.float16)
    got = cache.attend((q * 0.1).to(torch.bfloat16), table, torch.tensor([128], dtype=torch.int32, device="cuda"))
    _check(got, _plain((q * 0.1).to(torch.bfloat16), cache, table, [128], [0, 1], 0.125))
    small = _normal((128, 1, 64), 5) * 1e-5
    small[::3] = 0
    cache.append(_normal((128, 1, 64), 3), small, torch.arange(128, device="cuda"))
    got = cache.attend(q.to(torch.bfloat16), table, torch.tensor([128], dtype=torch.int32, device="cuda"))
    out, lse, bound, slack = _plain(q.to(torch.bfloat16), cache, table, [128], [0, 1], 0.125)
    assert ((got.double() - out).abs() <= 2.0**-8 * out.abs() + (2.0**-9 + 2 * slack.unsqueeze(-1)) * bound).all()


@pytest.mark.parametrize("rows", [None, [4, 1, 70]])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_does_not_matter(rows, dim):
    """NaN, infinite and huge scales in every slot that no row sees leave the results bit for bit the same."""
    lengths, page = [33, 16, 200], 16
    cache, table, query, got = _run(dim, 2, 4, page, "f16", lengths, rows=rows, window=50, seed=4)
    used = torch.zeros((cache.num_pages, page), dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        first = max(0, n - 50 - (0 if rows is None else rows[b] - 1))
        j = torch.arange(first, n, device="cuda")
        used[table[b].long()[j // page], j % page] = True
    offsets = None if rows is None else torch.tensor([0] + np.cumsum(rows).tolist(), dtype=torch.int32, device="cuda")
    for bad in (float("nan"), float("inf"), 3e38, -float("inf")):
        for t in (cache.k_scales, cache.v_scales):
            t.copy_(torch.where(used.unsqueeze(1), t, bad))
        again = cache.attend(query, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), query_offsets=offsets,
                             max_query_tokens=None if rows is None else max(rows), window=50)
        assert torch.equal(got, again)


@pytest.mark.parametrize("which", ["key", "value"])
def test_causal_rows_before_a_vector_that_is_not_finite(which):
    """Rows that see such a token are NaN; earlier rows of the same sequence are unharmed."""
    cache = _random_cache(8, 16, 1, 128, seed=6)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
    lengths, offsets = torch.tensor([128], dtype=torch.int32, device="cuda"), torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    q = _normal((100, 4, 128), 1, torch.bfloat16)
    clean = cache.attend(q, table, lengths, query_offsets=offsets, max_query_tokens=100)
    (cache.k_scales if which == "key" else cache.v_scales)[90 // 16, 0, 90 % 16] = float("nan")
    got = cache.attend(q, table, lengths, query_offsets=offsets, max_query_tokens=100)
    first = 90 - 28  # row i is at position 28 + i
    assert torch.equal(got[:first], clean[:first])
    assert torch.isnan(got[first:]).all()


def test_pages_outside_the_cache_are_not_seen():
    cache = _random_cache(6, 16, 2, 64, seed=8)
    table = torch.tensor([[0, 6, 2, -1, 4], [1 << 30, -5, 6, 99, 7]], dtype=torch.int32, device="cuda")
    lengths = [75, 80]
    q = _normal((2, 4, 64), 3, torch.float16)
    got, lse = cache.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), return_lse=True)
    _check(got, _plain(q, cache, table, lengths, [0, 1, 2], 0.125), lse)
    assert not got[1].any() and torch.isinf(lse[1]).all()


def test_lengths_and_offsets_are_held_to_what_exists():
    """A length past the table means the table's end; a negative one is zero; rows past the query are dropped."""
    cache = _random_cache(4, 16, 1, 64, seed=2)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    q = _normal((2, 2, 64), 5, torch.bfloat16)
    got = cache.attend(q, table, torch.tensor([1 << 30, -7], dtype=torch.int32, device="cuda"))
    _check(got, _plain(q, cache, table, [32, 0], [0, 1, 2], 0.125))
    offsets = torch.tensor([0, 1, 900], dtype=torch.int32, device="cuda")
    got = cache.attend(q, table, torch.tensor([20, 30], dtype=torch.int32, device="cuda"), query_offsets=offsets,
                       max_query_tokens=50)
    _check(got, _plain(q, cache, table, [20, 30], [0, 1, 2], 0.125))


def test_shared_and_repeated_pages():
    """Two sequences with a common prefix, and a table that names a page twice."""
    cache = _random_cache(5, 32, 2, 128, seed=12)
    table = torch.tensor([[3, 1, 0], [3, 1, 4], [2, 2, 2]], dtype=torch.int32, device="cuda")
    lengths = [80, 96, 70]
    q = _normal((3, 8, 128), 3, torch.bfloat16)
    got = cache.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    _check(got, _plain(q, cache, table, lengths, [0, 1, 2, 3], 128**-0.5))


def test_strided_query_and_tables():
    """Queries as a slice of a fused projection, heads before rows, tables and lengths as views."""
    page, lengths = 16, [40, 100]
    cache, table, query, got = _run(128, 2, 4, page, "bf16", lengths, rows=[3, 20], seed=15)
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 3, 23], dtype=torch.int32, device="cuda")
    wide = torch.zeros((23, 8 * 128 + 3), dtype=torch.bfloat16, device="cuda")
    wide[:, 1:-2] = query.flatten(1)
    spread = torch.full((2, 3 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    spread[:, ::3] = table
    long_lengths = torch.stack((length, length + 1), dim=1)[:, 0]
    for q in (wide[:, 1:-2].unflatten(1, (8, 128)), query.transpose(0, 1).contiguous().transpose(0, 1),
              query.transpose(1, 2).contiguous().transpose(1, 2)):
        again = cache.attend(q, spread[:, ::3], long_lengths, query_offsets=offsets, max_query_tokens=20)
        assert torch.equal(again, got)


def test_results_repeat_and_join_by_lse():
    """The same call gives the same bits; two halves of a context join to the whole by their log-sum-exp."""
    lengths = [64 * 16]
    cache, table, query, got = _run(128, 2, 4, 64, "f16", lengths, seed=20)
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    assert torch.equal(cache.attend(query, table, length), got)
    half = torch.tensor([512], dtype=torch.int32, device="cuda")
    (a, la), (b, lb) = (cache.attend(query, t, half, return_lse=True) for t in (table[:, :8], table[:, 8:16]))
    w = torch.softmax(torch.stack((la, lb)), dim=0).unsqueeze(-1)
    joined = w[0] * a.float() + w[1] * b.float()
    assert (joined - got.float()).abs().max() <= 2.0**-9 * got.float().abs().max()


def test_offsets_past_32_bits():
    """Pages whose vectors lie past 4 GB of codes and 2^31 dimensions."""
    page, heads, dim = 1024, 8, 128
    pages = 9000  # 4.7 GB of codes for keys, as much for values
    cache = m.Int4KVCache(pages, page, heads, dim)
    slots = torch.arange((pages - 2) * page, pages * page, device="cuda")
    k, v = _normal((2 * page, heads, dim), 1, torch.bfloat16), _normal((2 * page, heads, dim), 2, torch.bfloat16)
    cache.append(k, v, slots)
    assert cache.k_codes[-1, -1, -1].any() and not cache.k_codes[: pages - 2].any()
    small = m.Int4KVCache(2, page, heads, dim)
    near = torch.arange(2 * page, device="cuda")
    small.append(k, v, near)
    for far_x, near_x in zip(cache.read(slots), small.read(near)):
        assert torch.equal(far_x, near_x)
    for rows in (1, 200):
        q = _normal((rows, 16, dim), 3, torch.bfloat16)
        offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        length = torch.tensor([2 * page - 5], dtype=torch.int32, device="cuda")
        far = cache.attend(q, torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device="cuda"), length,
                           query_offsets=offsets, max_query_tokens=rows)
        here = small.attend(q, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), length, query_offsets=offsets,
                            max_query_tokens=rows)
        assert torch.equal(far, here)


def test_other_streams_and_graphs():
    """On a stream of its own, and replayed from a captured graph with new inputs in place."""
    lengths = [300, 5000]
    cache, table, query, got = _run(128, 2, 4, 16, "bf16", lengths, seed=30)
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    slots = cache.slots(table, torch.tensor([0, 1], device="cuda"), length - 1)
    keys = _normal((2, 2, 128), 77, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        results = [cache.attend(query, table, length) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(r, got) for r in results)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(keys, keys, slots)
        captured = cache.attend(query, table, length)
    keys.copy_(_normal((2, 2, 128), 78, torch.bfloat16))
    length.copy_(torch.tensor([299, 4000], dtype=torch.int32))
    slots.copy_(cache.slots(table, torch.tensor([0, 1], device="cuda"), length - 1))
    graph.replay()
    want = _plain(query, cache, table, [299, 4000], [0, 1, 2], 128**-0.5)
    _check(captured, want)
    back = cache.read(slots, dtype=torch.float32)[0]
    _, scales, codes = _packed(keys)
    np.testing.assert_array_equal(back.cpu().numpy().reshape(-1, 128), codes * scales[:, None])


def test_nothing_to_do():
    cache = m.Int4KVCache(2, 16, 2, 64)
    none = torch.zeros((0,), dtype=torch.int32, device="cuda")
    table = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    assert cache.attend(_normal((0, 4, 64), 1, torch.float16), table, none).shape == (0, 4, 64)
    q = _normal((3, 4, 64), 1, torch.float16)
    no_pages = torch.zeros((3, 0), dtype=torch.int32, device="cuda")
    got, lse = cache.attend(q, no_pages, torch.tensor([5, 0, 1], dtype=torch.int32, device="cuda"), return_lse=True)
    assert not got.any() and torch.isinf(lse).all()


# --------------------------------------------------------------------------- refusals

def test_refusals():
    for kw, text in (((4, 24, 2, 128), "page_size"), ((4, 8, 2, 128), "page_size"), ((4, 16, 2, 96), "head_dim"),
                     ((0, 16, 2, 64), "positive"), ((4, 16, 0, 64), "positive")):
        with pytest.raises(ValueError, match=text):
            m.Int4KVCache(*kw)
    with pytest.raises(ValueError, match="CUDA"):
        m.Int4KVCache(1, 16, 1, 64, device="cpu")
    cache = m.Int4KVCache(4, 16, 2, 64)
    raw = torch.zeros(4 * 2 * 16 * 32 + 1, dtype=torch.uint8, device="cuda")[1:].view(4, 2, 16, 32)
    with pytest.raises(ValueError, match="16-byte aligned"):
        m.Int4KVCache.from_tensors(raw, cache.k_scales, cache.v_codes, cache.v_scales)
    with pytest.raises(ValueError, match="shape"):
        m.Int4KVCache.from_tensors(cache.k_codes, cache.k_scales[:1], cache.v_codes, cache.v_scales)
    with pytest.raises(ValueError, match="dtype"):
        m.Int4KVCache.from_tensors(cache.k_codes, cache.k_scales.half(), cache.v_codes, cache.v_scales)
    with pytest.raises(ValueError, match="contiguous"):
        m.Int4KVCache.from_tensors(cache.k_codes.transpose(0, 1).contiguous().transpose(0, 1), cache.k_scales, cache.v_codes, cache.v_scales)
    x, slots = _normal((3, 2, 64), 1), torch.arange(3, device="cuda")
    for args, error, text in (((x.cpu(), x, slots), ValueError, "must be on"), ((x, x[:2], slots), ValueError, "same number"),
                              ((x, x.half(), slots), ValueError, "same dtype"), ((x.double(), x.double(), slots), ValueError, "dtype"),
                              ((x, x, slots.int()), ValueError, "dtype"), ((x[:, :1], x, slots), ValueError, "shape"),
                              ((x[..., :32], x, slots), ValueError, "shape"), ((x, x, [0, 1, 2]), TypeError, "tensor")):
        with pytest.raises(error, match=text):
            cache.append(*args)
    with pytest.raises(ValueError, match="dtype"):
        cache.read(slots, dtype=torch.float64)
    with pytest.raises(ValueError, match="contiguous"):
        cache.read(slots, out=(x[:2].half(), x[:2].half()))
    q = _normal((2, 4, 64), 2, torch.float16)
    table = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    length = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for args, kw, text in (((q.float(), table, length), {}, "fp16 or bf16"), ((q[:, :3], table, length), {}, "multiple"),
                           ((q[..., :32], table, length), {}, "shape"), ((q, table.long(), length), {}, "dtype"),
                           ((q, table, length.long()), {}, "dtype"), ((q, table[:1], length), {}, "batch"),
                           ((q[:1], table, length), {}, "one row per sequence"), ((q, table.cpu(), length), {}, "must be on"),
                           ((q, table, length), {"max_query_tokens": 2}, "query_offsets"),
                           ((q, table, length), {"query_offsets": offsets[:2]}, "batch \\+ 1"),
                           ((q, table, length), {"query_offsets": offsets, "max_query_tokens": -1}, "negative"),
                           ((q, table, length), {"window": 0}, "window"), ((q, table, length), {"window": 5, "causal": False}, "window"),
                           ((q, table, length), {"scale": 0.0}, "scale"), ((q, table, length), {"scale": float("nan")}, "scale"),
                           ((q, table, length), {"scale": float("inf")}, "scale"),
                           ((q, table, length), {"out": q[:1]}, "out"), ((q, table, length), {"out": q.bfloat16()}, "dtype")):
        with pytest.raises(ValueError, match=text):
            cache.attend(*args, **kw)
