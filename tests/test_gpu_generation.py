"""The cache and the weights together, as a reader model uses them, and the cache attention's ways against each other."""

import sys
from pathlib import Path

import pytest

import maxsim_b200 as m
from maxsim_b200 import _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

sys.path.insert(0, str(Path(__file__).resolve().parent))

import test_gpu_kv4 as kv4  # noqa: E402
import test_gpu_w4 as w4  # noqa: E402
from test_gpu_kv4 import _check, _normal, _plain, _random_cache, _tables  # noqa: E402


@pytest.fixture(params=[0, 1, 2], ids=["auto", "few", "many"])
def engine(request):
    """The attention kernel: by size, that for few rows, that for many."""
    _lib.set_option("kv4_engine", request.param)
    yield request.param
    _lib.set_option("kv4_engine", 0)


# The cache's tests once more on each kernel.
@pytest.mark.parametrize("dtype,dim", [("f16", 64), ("bf16", 128), ("f16", 128), ("bf16", 256)])
@pytest.mark.parametrize("shared", [1, 4, 7])
@pytest.mark.parametrize("window", [None, 1, 33, 200])
def test_ragged_rows(engine, dtype, dim, shared, window):
    kv4.test_ragged_rows(dtype, dim, shared, window)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,length", [(1, 1), (1, 300), (64, 64), (127, 500), (128, 128), (129, 1000), (300, 1111)])
@pytest.mark.parametrize("shared", [1, 4, 9])
def test_chunks(engine, dim, rows, length, shared):
    kv4.test_chunks(dim, rows, length, shared)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_pages(engine, page):
    kv4.test_page_sizes(page)


@pytest.mark.parametrize("rows", [None, [4, 1, 70]])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_does_not_matter(engine, rows, dim):
    kv4.test_what_is_not_seen_does_not_matter(rows, dim)


@pytest.mark.parametrize("which", ["key", "value"])
def test_vectors_that_are_not_finite(engine, which):
    kv4.test_causal_rows_before_a_vector_that_is_not_finite(which)


def test_other_cases_of_the_cache(engine):
    for rows in (None, [3, 1, 20], [200, 1, 64]):
        kv4.test_without_causal(rows)
    for window in (1, 64, 100000):
        kv4.test_window_of_one_token(window)
    for size in (1e-30, 1e-8, 1e8, 1e30):
        kv4.test_range_of_bf16(size)
    kv4.test_peaked_scores_and_rising_maxima()
    kv4.test_values_of_very_different_sizes()
    kv4.test_pages_outside_the_cache_are_not_seen()
    kv4.test_lengths_and_offsets_are_held_to_what_exists()
    kv4.test_shared_and_repeated_pages()
    kv4.test_strided_query_and_tables()
    kv4.test_results_repeat_and_join_by_lse()
    kv4.test_nothing_to_do()


def test_offsets_past_32_bits(engine):
    kv4.test_offsets_past_32_bits()


@pytest.mark.parametrize("batch,heads,rows,length", [(2, 16, 70, 300), (40, 8, 33, 150), (3, 8, 260, 900)])
def test_sizes_that_choose_the_kernel_for_many_rows(batch, heads, rows, length):
    kv4._run(128, heads, 4, 32, "bf16", [length - 3 * b for b in range(batch)], rows=[max(1, rows - b) for b in range(batch)])


def test_example_answers_from_what_it_found():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import answer_from_retrieved as example

    before = _lib.launch_count()
    wanted, found, answer = example.main(layers=2, tokens=4)
    assert (found[:, 0] == wanted).all()
    assert answer.shape == (3, 4) and int(answer.min()) >= 0 and int(answer.max()) < 1000
    # per forward pass and layer: four products, an append, an attention; a product per token for the words
    assert _lib.launch_count() - before >= 5 * 2 * 6 + 4
    assert torch.equal(example.main(layers=2, tokens=4)[2], answer)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("split", [1, 7, 40])
def test_chunks_and_single_tokens_agree(engine, dim, split):
    """A prompt attended to in one chunk, in pieces, or a token at a time gives the same rows (to the rounding of
    probabilities and outputs)."""
    length, heads, shared = 200, 2, 4
    cache = _random_cache(16, 16, heads, dim, seed=dim)
    table = _tables([length], 16, 16, extra=0)
    q = _normal((length, heads * shared, dim), 3, torch.bfloat16)

    def rows(lo, hi):
        return cache.attend(q[lo:hi], table, torch.tensor([hi], dtype=torch.int32, device="cuda"),
                            query_offsets=torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda"), max_query_tokens=hi - lo)

    whole = rows(0, length)
    pieces = torch.cat([rows(lo, min(length, lo + split)) for lo in range(0, length, split)])
    want = _plain(q, cache, table, [length], [0, length], dim**-0.5)
    _check(whole, want)
    _check(pieces, want)


@pytest.mark.parametrize("rows", [20, 100])
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_many_rows_far_outside_fp16(engine, rows, size):
    """Queries, keys and values whose sizes fp16 does not hold, with many rows a sequence."""
    cache = m.Int4KVCache(12, 16, 2, 128)
    every = torch.arange(12 * 16, device="cuda")
    cache.append(_normal((192, 2, 128), 3) / size, _normal((192, 2, 128), 2) * size, every)
    table = _tables([150], 16, 12)
    q = (_normal((rows, 8, 128), 4) * size).to(torch.bfloat16)
    offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    got = cache.attend(q, table, torch.tensor([150], dtype=torch.int32, device="cuda"), query_offsets=offsets, max_query_tokens=rows)
    out, lse, bound, slack = _plain(q, cache, table, [150], [0, rows], 128**-0.5)
    assert ((got.double() - out).abs() <= 2.0**-8 * out.abs() + (2.0**-10 + 2 * slack.unsqueeze(-1)) * bound).all()


@pytest.mark.parametrize("rows", [None, 70])
@pytest.mark.parametrize("growing", [True, False])
def test_value_sizes_and_scores_that_run_apart(engine, rows, growing):
    """Value sizes over nine decades along the sequence, with scores that rise or fall: references move often."""
    n = 640
    cache = m.Int4KVCache(40, 16, 1, 128)
    ramp = torch.linspace(-1, 1, n, device="cuda") * (1 if growing else -1)
    direction = _normal((1, 1, 128), 4)
    k = direction * (3 * ramp).view(-1, 1, 1) + _normal((n, 1, 128), 5, scale=0.1)
    v = _normal((n, 1, 128), 6) * (10.0 ** (4.5 * ramp)).view(-1, 1, 1)
    cache.append(k, v, torch.arange(n, device="cuda"))
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40)
    count = rows or 1
    q = (direction * 2 + _normal((count, 4, 128), 7)).to(torch.bfloat16)
    got = cache.attend(q, table, torch.tensor([n], dtype=torch.int32, device="cuda"),
                       query_offsets=None if rows is None else torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                       max_query_tokens=rows)
    _check(got, _plain(q, cache, table, [n], [0, count], 128**-0.5))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 3, 90])
def test_outputs_and_queries_off_16_bytes(engine, dim, rows):
    """A caller's output that starts 2 bytes off, and queries that do, give the aligned call's bits."""
    cache = _random_cache(10, 16, 2, dim, seed=1)
    table = _tables([140], 16, 10, extra=0)
    q = _normal((rows, 6, dim), 2, torch.float16)
    length = torch.tensor([140], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    want = cache.attend(q, table, length, query_offsets=offsets, max_query_tokens=rows)
    room = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")
    out = room[1:].view(q.shape)
    assert cache.attend(q, table, length, query_offsets=offsets, max_query_tokens=rows, out=out) is not None
    assert torch.equal(out, want)
    off = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    off.copy_(q)
    assert torch.equal(cache.attend(off, table, length, query_offsets=offsets, max_query_tokens=rows), want)


@pytest.mark.parametrize("batch", [1, 31, 32, 33, 128, 129, 300])
def test_numbers_of_sequences(batch):
    """The search of the work line by warps and by blocks, sequences without rows or tokens among them."""
    lengths = [(37 * i) % 400 for i in range(batch)]
    rows = [(i * 5) % 4 for i in range(batch)]
    rows[0] = 1
    page = 16
    pages = sum(-(-n // page) for n in lengths) + 1
    cache = _random_cache(pages, page, 2, 64, seed=batch)
    table = _tables(lengths, page, pages, extra=600, seed=batch)  # a wide table: contexts could be long
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    q = _normal((starts[-1], 6, 64), 2, torch.bfloat16)
    got, lse = cache.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                            query_offsets=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_query_tokens=3, return_lse=True)
    _check(got, _plain(q, cache, table, lengths, starts, 0.125), lse)


def test_calls_on_two_streams_at_once():
    """Two streams attend over one cache at the same time: workspaces are each call's own."""
    cache = _random_cache(700, 64, 4, 128, seed=5)
    lengths = [20000, 15000]
    table = _tables(lengths, 64, 700)
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    qs = [_normal((2, 16, 128), i, torch.bfloat16) for i in range(2)]
    want = [cache.attend(q, table, length) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(cache.attend(q, table, length))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


def test_more_query_tokens_announced_than_there_are(engine):
    cache = _random_cache(22, 16, 2, 128, seed=3)
    table = torch.arange(22, dtype=torch.int32, device="cuda").flip(0).expand(2, -1)
    query = _normal((7, 8, 128), 5, torch.bfloat16)
    lengths = torch.tensor([300, 41], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 5, 7], dtype=torch.int32, device="cuda")
    want = cache.attend(query, table, lengths, query_offsets=offsets, max_query_tokens=7)
    got = cache.attend(query, table, lengths, query_offsets=offsets, max_query_tokens=(1 << 31) - 1)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(3552, 200), (3551, 72), (5001, 328), (9600, 136)])
@pytest.mark.parametrize("rows", [2, 8, 11, 16, 20, 32])
def test_product_of_many_weight_rows(dtype, group, n, k, rows):
    packed, scales, w = w4._codes(n, k, group, seed=n + k)
    x = _normal((rows, k), rows, kv4.DTYPES[dtype])
    w4._check(m.Int4Linear(packed, scales, group_size=group)(x), x, w, None, group)
