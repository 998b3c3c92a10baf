"""Products of few rows with 4-bit weights, against plain arithmetic in 64 bits."""

import pytest

import maxsim_b200 as m

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _normal(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _codes(n, k, group, seed):
    """Codes with every value -7 .. 7 and scales of several sizes: packed bytes, bf16 scales, 64-bit weights."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = torch.randint(-7, 8, (n, k), generator=g, device="cuda", dtype=torch.int16)
    scales = torch.exp(_normal((n, -(-k // group)), seed + 1)).to(torch.bfloat16) * 0.02
    packed = ((c[:, 0::2] & 15) | ((c[:, 1::2] & 15) << 4)).to(torch.uint8)
    return packed, scales, c.double() * scales.double().repeat_interleave(group, dim=1)[:, :k]


def _check(got, x, w, bias, group):
    """Products of a code and an input are exact in fp32; a sum passes at most k / 16 + k / group + 48 roundings
    of 24 bits (a cut rather than a rounding allowed), each of at most sum |x w|; then one rounding to the output."""
    y = x.double() @ w.t()
    if bias is not None:
        y = y + bias.double()
    k = w.shape[1]
    # Per group the sum is of x * code, scaled after: its size is that of the group's sum |x code| * scale.
    size = x.double().abs() @ w.abs().t() + (0 if bias is None else bias.double().abs())
    eps = 2.0**-8 if got.dtype == torch.bfloat16 else 2.0**-10
    limit = eps * y.abs() + size * (k / 16 + k / group + 48) * 2.0**-23 + 2.0**-24
    off = (got.double() - y).abs()
    assert got.shape == y.shape and (off <= limit).all(), f"worst {(off / limit).max().item():.3g} of the bound"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 8), (15, 64), (16, 128), (17, 136), (100, 1000), (256, 2048), (1111, 2080), (33, 40)])
@pytest.mark.parametrize("rows", [1, 3, 8, 9, 17])
def test_product(dtype, group, n, k, rows):
    packed, scales, w = _codes(n, k, group, seed=n + k)
    bias = _normal((n,), 5, DTYPES[dtype]) if (n + rows) % 2 else None
    x = _normal((rows, k), rows, DTYPES[dtype])
    _check(m.Int4Linear(packed, scales, group_size=group, bias=bias)(x), x, w, bias, group)


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 7, 8, 12, 16, 24, 31, 32, 33, 64, 100, 257])
def test_numbers_of_rows(rows):
    packed, scales, w = _codes(300, 1224, 64, seed=1)
    x = _normal((rows, 1224), rows, torch.bfloat16)
    _check(m.Int4Linear(packed, scales, group_size=64)(x), x, w, None, 64)


@pytest.mark.parametrize("n,k,rows,group", [(4096, 4096, 1, 128), (16384, 8192, 16, 64), (64, 65536, 2, 128), (70000, 64, 1, 32)])
def test_large(n, k, rows, group):
    packed, scales, w = _codes(n, k, group, seed=n)
    x = _normal((rows, k), 3, torch.bfloat16)
    _check(m.Int4Linear(packed, scales, group_size=group)(x), x, w, None, group)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_inputs_with_a_common_offset(dtype):
    """Inputs far from zero: what the codes' storage adds to them must not cost digits."""
    packed, scales, w = _codes(64, 512, 128, seed=2)
    x = _normal((4, 512), 3, DTYPES[dtype]) + 20
    _check(m.Int4Linear(packed, scales)(x), x, w, None, 128)


def test_views_shapes_and_out():
    packed, scales, w = _codes(50, 128, 32, seed=3)
    linear = m.Int4Linear(packed, scales, group_size=32)
    base = _normal((6, 4 * 128 + 3), 4, torch.float16)
    for x in (base[:, 1:129], base[::2, :128], base[:, : 2 * 128 : 2], _normal((1, 128), 5, torch.float16).expand(3, 128)):
        want = linear(x.contiguous())
        _check(want, x, w, None, 32)
        assert torch.equal(linear(x), want)
    x = _normal((2, 3, 128), 6, torch.float16)
    got = linear(x)
    assert got.shape == (2, 3, 50) and torch.equal(got.view(6, 50), linear(x.view(6, 128)))
    assert torch.equal(linear(x[0, 0]), linear(x[0, :1])[0])
    out = torch.empty((2, 3, 50), dtype=torch.float16, device="cuda")
    assert linear(x, out=out) is out and torch.equal(out, got)
    assert linear(x[:0]).shape == (0, 3, 50)


@pytest.mark.parametrize("rows", [1, 9])
def test_infinities_and_nan_stay_in_their_row(rows):
    packed, scales, w = _codes(40, 256, 64, seed=4)
    linear = m.Int4Linear(packed, scales, group_size=64)
    x = _normal((rows + 1, 256), 7, torch.bfloat16)
    clean = linear(x)
    x[rows, 17] = float("nan")
    got = linear(x)
    assert torch.equal(got[:rows], clean[:rows]) and torch.isnan(got[rows]).all()


def test_from_weight():
    """Scales are bf16(max / 7), codes the nearest to the rounded scale; zero groups and short last groups."""
    weight = _normal((30, 200), 8, scale=0.05)
    weight[3, 64:128] = 0
    linear = m.Int4Linear.from_weight(weight, group_size=64)
    padded = torch.nn.functional.pad(weight, (0, 56)).view(30, 4, 64)
    scale = (padded.abs().amax(-1) / 7).bfloat16().float()
    scale[scale == 0] = 1
    w = (torch.round(padded / scale.unsqueeze(-1)).clamp(-7, 7).double() * scale.double().unsqueeze(-1)).view(30, 256)[:, :200]
    x = _normal((5, 200), 9, torch.bfloat16)
    _check(linear(x), x, w, None, 64)
    # the weight itself is within half a code step (and the rounding of the scale at the ends of the range)
    assert ((w - weight.double()).abs() <= 0.5 * scale.double().repeat_interleave(64, 1)[:, :200] * 1.06).all()


def test_results_repeat_on_streams_and_graphs():
    packed, scales, w = _codes(2000, 4096, 128, seed=5)
    linear = m.Int4Linear(packed, scales)
    x = _normal((3, 4096), 1, torch.bfloat16)
    got = linear(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        results = [linear(x) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(r, got) for r in results)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = linear(x)
    x.copy_(_normal((3, 4096), 2, torch.bfloat16))
    graph.replay()
    assert torch.equal(captured, linear(x))


def test_refusals():
    packed, scales, _ = _codes(16, 64, 32, seed=6)
    for kw, text in ((dict(codes=packed.cpu()), "CUDA"), (dict(codes=packed.short()), "dtype"), (dict(codes=packed[:, :30]), "multiple of 8"),
                     (dict(codes=packed[:0]), "positive"), (dict(scales=scales.float()), "dtype"), (dict(scales=scales[:, :1]), "shape"),
                     (dict(group_size=48), "group"), (dict(bias=torch.zeros(16, device="cuda")), "dtype"),
                     (dict(bias=torch.zeros(15, device="cuda", dtype=torch.float16)), "bias")):
        args = {"codes": packed, "scales": scales, "group_size": 32, **kw}
        with pytest.raises(ValueError, match=text):
            m.Int4Linear(args.pop("codes"), args.pop("scales"), **args)
    linear = m.Int4Linear(packed, scales, group_size=32, bias=torch.zeros(16, device="cuda", dtype=torch.float16))
    x = _normal((2, 64), 1, torch.float16)
    for bad, kw, text in ((x.float(), {}, "fp16 or bf16"), (x[:, :32], {}, "shape"), (x.cpu(), {}, "must be on"),
                          (x.bfloat16(), {}, "bias"), (x, {"out": x[:, :16]}, "contiguous"), (x, {"out": x.bfloat16()}, "dtype")):
        with pytest.raises(ValueError, match=text):
            linear(bad, **kw)
    for bad, text in ((torch.zeros((4, 12), device="cuda"), "multiple of 8"), (torch.full((2, 64), float("inf"), device="cuda"), "finite"),
                      (torch.zeros((64,), device="cuda"), "shape")):
        with pytest.raises(ValueError, match=text):
            m.Int4Linear.from_weight(bad)
    with pytest.raises(ValueError, match="group_size"):
        m.Int4Linear.from_weight(torch.zeros((4, 64), device="cuda"), group_size=16)
