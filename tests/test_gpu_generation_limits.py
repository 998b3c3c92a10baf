"""The cache attention and the weight products where their arguments or their data reach a limit."""

import ctypes
import sys
from pathlib import Path

import pytest

import maxsim_b200 as m
from maxsim_b200 import _lib
from maxsim_b200._lib import check, lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

sys.path.insert(0, str(Path(__file__).resolve().parent))

from test_gpu_kv4 import _check, _normal, _plain, _random_cache, _tables  # noqa: E402


@pytest.fixture(params=[0, 1, 2], ids=["auto", "few", "many"])
def engine(request):
    """The attention kernel: by size, that for few rows, that for many."""
    _lib.set_option("kv4_engine", request.param)
    yield request.param
    _lib.set_option("kv4_engine", 0)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# --------------------------------------------------------------------------- the C entry's workspace

def _c_attend(cache, query, table, lengths, workspace, workspace_bytes, out):
    """One row a sequence through the C entry, with the caller's workspace."""
    c = _lib.Kv4Cache(cache.k_codes.data_ptr(), cache.k_scales.data_ptr(), cache.v_codes.data_ptr(), cache.v_scales.data_ptr(),
                      cache.num_pages, cache.page_size, cache.num_kv_heads, cache.head_dim, 0)
    a = _lib.Kv4AttendArgs(query=query.data_ptr(), query_row_stride=query.stride(0), query_head_stride=query.stride(1),
                           rows=query.shape[0], page_table=table.data_ptr(), page_table_stride=table.stride(0),
                           lengths=lengths.data_ptr(), out=out.data_ptr(), workspace=workspace, workspace_bytes=workspace_bytes,
                           batch=table.shape[0], max_pages=table.shape[1], max_query_rows=1, heads=query.shape[1],
                           type=_lib.TYPE_F16, causal=1, scale=query.shape[2] ** -0.5)
    need = ctypes.c_int64()
    check(lib.msb_kv4_attend_workspace_bytes(ctypes.byref(c), ctypes.byref(a), ctypes.byref(need)))
    if workspace is not None:
        if workspace_bytes is None:
            a.workspace_bytes = need.value
        check(lib.msb_kv4_attend_device(ctypes.byref(c), ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
    return need.value


@pytest.mark.parametrize("batch", [1, 32, 33, 40, 300])
@pytest.mark.parametrize("pages_each", [1, 8, 9, 70])
def test_the_workspace_that_was_asked_for_is_all_that_is_written(batch, pages_each):
    """Memory past what msb_kv4_attend_workspace_bytes names keeps what it held; where it names nothing, all of it."""
    page, dim = 16, 64
    cache = _random_cache(pages_each * 2, page, 2, dim, seed=1)
    lengths = _ints(*[(7 * b) % (pages_each * page + 1) for b in range(batch)])
    table = torch.arange(pages_each, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    query = _normal((batch, 4, dim), 2, torch.float16)
    out = torch.zeros_like(query)
    need = _c_attend(cache, query, table, lengths, None, 0, out)
    room = torch.full((need + 8192,), 0x5A, dtype=torch.uint8, device="cuda")
    assert _c_attend(cache, query, table, lengths, room.data_ptr(), need, out) == need
    assert (room[need:] == 0x5A).all()
    if pages_each * page <= 128:
        assert need == 0
    assert torch.equal(out, cache.attend(query, table, lengths))


# --------------------------------------------------------------------------- windows

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 2, (1 << 31) - 100, 1 << 31, 1 << 62])
@pytest.mark.parametrize("wide", [0, 200])
def test_windows_of_any_size_where_rows_outnumber_tokens(engine, dim, window, wide):
    """A window as large as a number can be hides nothing: the bits of the call without one, in blocks of rows that all
    lie before the sequence's first token, that lie on both sides of it, and after."""
    lengths, rows, page = [200, 1, 0, 40, 70], [600, 290, 5, 43, 1], 16
    cache = _random_cache(24, page, 2, dim, seed=dim)
    table = _tables(lengths, page, 24, extra=1 + wide)
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    query = _normal((starts[-1], 6, dim), 3, torch.bfloat16)
    kw = dict(query_offsets=_ints(*starts), max_query_tokens=max(rows), return_lse=True)
    want, want_lse = cache.attend(query, table, _ints(*lengths), **kw)
    _check(want, _plain(query, cache, table, lengths, starts, dim**-0.5), want_lse)
    got, lse = cache.attend(query, table, _ints(*lengths), window=window, **kw)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


# --------------------------------------------------------------------------- announced rows

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("most", [1, 3, 20])
@pytest.mark.parametrize("wide", [0, 200])
@pytest.mark.parametrize("window", [None, 30])
def test_fewer_query_tokens_announced_than_there_are(engine, dim, most, wide, window):
    """Rows up to the announced number are those of the whole call, at their own positions; rows past it keep what the
    caller's output held."""
    lengths, starts, page = [40, 90, 25, 3], [0, 3, 33, 35, 45], 16
    cache = _random_cache(14, page, 2, dim, seed=dim)
    table = _tables(lengths, page, 14, extra=1 + wide)
    query = _normal((starts[-1], 6, dim), 3, torch.bfloat16)
    out = torch.full_like(query, 7.0)
    got, lse = cache.attend(query, table, _ints(*lengths), query_offsets=_ints(*starts), max_query_tokens=most, window=window,
                            return_lse=True, out=out)
    want = _plain(query, cache, table, lengths, starts, dim**-0.5, window=window)
    kept = torch.zeros(starts[-1], dtype=torch.bool, device="cuda")
    for lo, hi in zip(starts, starts[1:]):
        kept[lo : min(hi, lo + most)] = True
    _check(got[kept], [t[kept] for t in want], lse[kept])
    assert (out[~kept] == 7.0).all()


def test_no_query_tokens_announced_where_there_are_some():
    cache = _random_cache(4, 16, 2, 64, seed=1)
    q = _normal((3, 4, 64), 1, torch.float16)
    table, lengths = _ints(0, 1, 2, 3).view(2, 2), _ints(20, 30)
    with pytest.raises(ValueError, match="max_query"):
        cache.attend(q, table, lengths, query_offsets=_ints(0, 1, 3), max_query_tokens=0)
    assert cache.attend(q[:0], table, lengths, query_offsets=_ints(0, 0, 0), max_query_tokens=0).shape == (0, 4, 64)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch,wide", [(3, 0), (3, 300), (40, 0), (40, 300), (140, 300)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_without_a_sequence_are_zero(engine, dim, batch, wide, dtype):
    """In an output of the call's own, rows before the first offset and after the last are zeros with a log-sum-exp of
    -inf, rows past the announced number NaN; a caller's output keeps what it held there."""
    page, most = 16, 2
    lengths = [(29 * b) % 60 for b in range(batch)]
    starts = [5]
    for b in range(batch):
        starts.append(starts[-1] + b % 4)
    rows = starts[-1] + 37
    pages = sum(-(-n // page) for n in lengths) + 1
    cache = _random_cache(pages, page, 2, dim, seed=batch)
    table = _tables(lengths, page, pages, extra=1 + wide)
    query = _normal((rows, 6, dim), 3, dtype)
    past = torch.zeros(rows, dtype=torch.bool, device="cuda")
    kept = past.clone()
    for lo, hi in zip(starts, starts[1:]):
        kept[lo : min(hi, lo + most)] = True
        past[min(hi, lo + most) : hi] = True
    nobody = ~(kept | past)
    args = (query, table, _ints(*lengths))
    kw = dict(query_offsets=_ints(*starts), max_query_tokens=most)
    for _ in range(3):
        held = torch.full((rows, 6, dim), 7.0, dtype=dtype, device="cuda"), torch.full((rows, 6), 7.0, device="cuda")
        del held  # memory of these sizes is the allocator's next answer, and not zero
        got, lse = cache.attend(*args, return_lse=True, **kw)
        assert not got[nobody].any() and (lse[nobody] == -torch.inf).all()
        assert torch.isnan(got[past]).all() and torch.isnan(lse[past]).all()
    out = torch.full_like(query, 7.0)
    _, lse = cache.attend(*args, out=out, return_lse=True, **kw)
    assert (out[~kept] == 7.0).all() and torch.equal(out[kept], got[kept])
    assert (lse[~kept] == -torch.inf).all()


def test_no_sequence_has_rows(engine):
    cache = _random_cache(4, 16, 2, 64, seed=1)
    for batch, offsets in ((2, _ints(0, 0, 0)), (2, _ints(9, 9, 9)), (0, _ints(0))):
        q = _normal((9, 4, 64), 1, torch.float16)
        torch.full_like(q, 7.0)
        got, lse = cache.attend(q, _ints(0, 1, 2, 3).view(2, 2)[:batch], _ints(20, 30)[:batch], query_offsets=offsets,
                                return_lse=True)
        assert not got.any() and (lse == -torch.inf).all()


# --------------------------------------------------------------------------- sizes of values

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("exponent", [-112, -120, None])
@pytest.mark.parametrize("tokens", [4096, 20000])
def test_values_so_small_that_weights_grow(engine, dim, rows, exponent, tokens):
    """Thousands of like tokens whose value scales are 2^-112 or less (or zero): sums of weights stay finite.

    Outputs: the bound of `_check` without its absolute part.  Log-sum-exp: fp32 sums of at most 20,000 terms in parts,
    1e-5."""
    page = 64
    pages = -(-tokens // page)
    cache = _random_cache(pages, page, 1, dim, seed=2)
    cache.v_scales.fill_(0.0 if exponent is None else 2.0**exponent)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(1, -1)
    q = _normal((rows, 4, dim), 3, torch.bfloat16, 0.1)
    got, lse = cache.attend(q, table, _ints(tokens), query_offsets=_ints(0, rows), max_query_tokens=rows, return_lse=True)
    out, want_lse, bound, slack = _plain(q, cache, table, [tokens], [0, rows], dim**-0.5)
    assert ((lse.double() - want_lse).abs() <= slack + 1e-5 + 1e-6 * want_lse.abs()).all()
    assert ((got.double() - out).abs() <= 2.0**-8 * out.abs() + (2.0**-10 + 2 * slack.unsqueeze(-1)) * bound).all()


@pytest.mark.parametrize("rows", [1, 70])
def test_zero_scales_and_scores_that_rise(engine, rows):
    """Value scales of zero never raise a reference by their products: scores that rise by hundreds of powers of two
    along the sequence must not overflow their weights."""
    n, page = 640, 16
    cache = m.Int4KVCache(40, page, 1, 128)
    direction = _normal((1, 1, 128), 4)
    cache.append(direction * torch.linspace(-30, 30, n, device="cuda").view(-1, 1, 1), _normal((n, 1, 128), 6),
                 torch.arange(n, device="cuda"))
    cache.v_scales.zero_()
    cache.v_scales[0, 0, 3] = 1.0
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40)
    q = (direction * 2).expand(rows, 4, 128).to(torch.bfloat16)
    got, lse = cache.attend(q, table, _ints(n), query_offsets=_ints(0, rows), max_query_tokens=rows, return_lse=True)
    want = _plain(q, cache, table, [n], [0, rows], 128**-0.5)
    _check(got, want, lse)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("size", [1e-5, 1e-6, 1e-8, 1e-9, 1e-20])
@pytest.mark.parametrize("every", [2, 3, 40])
def test_zero_vectors_among_small_values(engine, dim, rows, size, every):
    """A vector of zeros is stored with scale 1, whatever its neighbours' sizes: it must not decide how the others'
    weights are held.  Bound: that of `_check` without its absolute part."""
    n, page = 300, 16
    cache = m.Int4KVCache(19, page, 1, dim)
    v = _normal((n, 1, dim), 5) * size
    v[1::every] = 0
    cache.append(_normal((n, 1, dim), 3), v, torch.arange(n, device="cuda"))
    table = torch.arange(19, dtype=torch.int32, device="cuda").view(1, -1)
    q = _normal((rows, 4, dim), 4, torch.bfloat16)
    got, lse = cache.attend(q, table, _ints(n), query_offsets=_ints(0, rows), max_query_tokens=rows, return_lse=True)
    out, want_lse, bound, slack = _plain(q, cache, table, [n], [0, rows], dim**-0.5)
    assert ((lse.double() - want_lse).abs() <= slack + 1e-5 + 1e-6 * want_lse.abs()).all()
    off, limit = (got.double() - out).abs(), 2.0**-8 * out.abs() + (2.0**-10 + 2 * slack.unsqueeze(-1)) * bound
    assert (off <= limit).all(), f"worst {(off / limit).max().item():.3g} of the bound"


def test_scales_of_one_that_are_not_zero_vectors(engine):
    """Ordinary vectors with a scale of exactly 1 keep their part."""
    cache = _random_cache(10, 16, 2, 128, seed=8)
    cache.v_scales[:, :, ::2] = 1.0
    table = _ints(*range(10)).view(1, 10)
    q = _normal((70, 8, 128), 4, torch.bfloat16)
    got, lse = cache.attend(q, table, _ints(150), query_offsets=_ints(0, 70), max_query_tokens=70, return_lse=True)
    _check(got, _plain(q, cache, table, [150], [0, 70], 128**-0.5), lse)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("size", [1e-37, 1e-35, 1e33, 1e35, 1e37])
def test_the_largest_and_smallest_queries(engine, dim, rows, size):
    """Queries near both ends of bf16 over keys near the other end: their scores are ordinary numbers."""
    n, page = 150, 16
    cache = m.Int4KVCache(10, page, 1, dim)
    cache.append(_normal((n, 1, dim), 3) / size, _normal((n, 1, dim), 5), torch.arange(n, device="cuda"))
    table = _ints(*range(10)).view(1, 10)
    q = (_normal((rows, 4, dim), 4) * size).to(torch.bfloat16)
    got, lse = cache.attend(q, table, _ints(n), query_offsets=_ints(0, rows), max_query_tokens=rows, return_lse=True)
    _check(got, _plain(q, cache, table, [n], [0, rows], dim**-0.5), lse)



@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("size", [1e33, 1e35, 1e37, 1e38])
def test_the_largest_finite_values(engine, dim, rows, size):
    """Values up to fp32's and bf16's largest numbers: outputs are finite where their averages are.  Scores lie close
    together, so no weight is far from the largest; bound: that of `_check` without its absolute part."""
    n, page = 150, 16
    cache = m.Int4KVCache(10, page, 1, dim)
    v = (_normal((n, 1, dim), 5) * size).clamp(-3e38, 3e38)
    cache.append(_normal((n, 1, dim), 3), v, torch.arange(n, device="cuda"))
    assert torch.isfinite(cache.v_scales[:9]).all()
    table = _ints(*range(10)).view(1, 10)
    q = _normal((rows, 4, dim), 4, torch.bfloat16, 0.1)
    got, lse = cache.attend(q, table, _ints(n), query_offsets=_ints(0, rows), max_query_tokens=rows, return_lse=True)
    out, want_lse, bound, slack = _plain(q, cache, table, [n], [0, rows], dim**-0.5)
    assert ((lse.double() - want_lse).abs() <= slack + 1e-5 + 1e-6 * want_lse.abs()).all()
    off, limit = (got.double() - out).abs(), 2.0**-8 * out.abs() + (2.0**-10 + 2 * slack.unsqueeze(-1)) * bound
    assert (off <= limit).all(), f"worst {(off / limit).max().item():.3g} of the bound"


# --------------------------------------------------------------------------- products

@pytest.mark.parametrize("rows", [65535 * 32, 65535 * 32 + 1, 65536 * 32 + 33])
def test_products_of_millions_of_rows(rows):
    """More row blocks than a grid's second dimension has: every row is the product that it is alone."""
    w = _normal((16, 64), 1, scale=0.1)
    linear = m.Int4Linear.from_weight(w, group_size=64)
    x = _normal((rows, 64), 2, torch.bfloat16)
    got = linear(x)
    for at in (0, 1 << 20, 65535 * 32 - 64, rows - 100):
        at = min(at, rows - 64)
        assert torch.equal(got[at : at + 64], linear(x[at : at + 64].clone()))


# --------------------------------------------------------------------------- outputs over inputs

def test_outputs_that_overlap_what_is_read_are_refused():
    """Blocks write while others read: a product into its own input, rows or heads of it, or a shifted view of it."""
    linear = m.Int4Linear.from_weight(_normal((64, 64), 1, scale=0.1), group_size=64)
    room = _normal((40, 64), 2, torch.bfloat16)
    x = room[:16]
    want = linear(x)
    for out in (x, room[8:24], room[15:31]):
        with pytest.raises(ValueError, match="overlap"):
            linear(x, out=out)
    assert torch.equal(linear(x, out=room[16:32]), want)  # the rows after
    wide = _normal((16, 128), 3, torch.bfloat16)
    want = linear(wide[1:2, 64:])
    assert torch.equal(linear(wide[1:2, 64:], out=wide[1:2, :64]), want)  # the other half of the row
    with pytest.raises(ValueError, match="overlap"):
        linear(wide[:, 64:], out=wide.flatten()[: 16 * 64].view(16, 64))
    odd = _normal((3 * 64 + 1,), 4, torch.bfloat16)[1:].view(3, 64)  # off 16 bytes: copied first, nothing to overlap
    want = linear(odd)
    assert torch.equal(linear(odd, out=odd), want)

    cache = _random_cache(8, 16, 2, 64, seed=1)
    rows = torch.zeros((20, 4, 64), dtype=torch.float16, device="cuda")
    rows.copy_(_normal((20, 4, 64), 5, torch.float16))
    table, lengths = _ints(*range(8)).view(1, 8), _ints(120)
    kw = dict(query_offsets=_ints(0, 10), max_query_tokens=10)
    for out in (rows[5:15], rows[9:19]):
        with pytest.raises(ValueError, match="overlap"):
            cache.attend(rows[:10], table, lengths, out=out, **kw)
    want = cache.attend(rows[:10], table, lengths, **kw)
    assert torch.equal(cache.attend(rows[:10], table, lengths, out=rows[10:], **kw), want)
    slots = torch.arange(4, device="cuda")
    pair = torch.zeros((6, 2, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        cache.read(slots, out=(pair[:4], pair[2:]))
    both = torch.zeros((8, 2, 64), dtype=torch.float16, device="cuda")
    keys, values = cache.read(slots, out=(both[:4], both[4:]))
    assert torch.equal(keys, cache.read(slots, dtype=torch.float16)[0]) and torch.equal(values, cache.read(slots, dtype=torch.float16)[1])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,length", [(1, 100), (5, 120), (3, 3000), (90, 3000)])
def test_attention_in_place_of_its_query(engine, dim, rows, length):
    """The output in the query's own memory: every block reads its rows before it writes them."""
    page = 16
    pages = -(-length // page)
    cache = _random_cache(pages, page, 2, dim, seed=dim)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(2, -1)
    query = _normal((2 * rows, 6, dim), 5, torch.bfloat16)
    kw = dict(query_offsets=_ints(0, rows, 2 * rows), max_query_tokens=rows)
    lengths = _ints(length, length - 1)
    want = cache.attend(query, table, lengths, **kw)
    assert torch.equal(cache.attend(query, table, lengths, out=query, **kw), want)


# --------------------------------------------------------------------------- gradients

def test_inputs_that_require_a_gradient_are_refused():
    """There is no backward pass: a result without a history must not pass for one with it."""
    linear = m.Int4Linear.from_weight(_normal((16, 64), 1), group_size=64)
    x = _normal((2, 64), 2, torch.bfloat16).requires_grad_()
    cache = _random_cache(4, 16, 2, 64, seed=1)
    table, lengths = _ints(0, 1, 2, 3).view(2, 2), _ints(20, 30)
    q = _normal((2, 4, 64), 3, torch.float16).requires_grad_()
    for call in (lambda: linear(x), lambda: cache.attend(q, table, lengths)):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            want = call()
        with torch.inference_mode():
            assert torch.equal(call(), want)
    assert torch.equal(linear(x.detach()), linear(x.detach() * 1))
    bias = torch.nn.Parameter(_normal((16,), 4, torch.bfloat16))
    m.Int4Linear.from_weight(_normal((16, 64), 1), group_size=64, bias=bias)(x.detach())  # held as a constant
    out = torch.zeros((2, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    pair = [torch.zeros((1, 2, 64), dtype=torch.float16, device="cuda", requires_grad=True) for _ in range(2)]
    for call in (lambda: linear(x.detach(), out=out), lambda: cache.attend(q.detach(), table, lengths, out=q),
                 lambda: cache.read(torch.zeros(1, dtype=torch.int64, device="cuda"), out=pair)):
        with pytest.raises(ValueError, match="gradient"):
            call()
