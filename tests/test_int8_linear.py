"""quantize_int8 and linear_int8 against their definitions in 64 bits.

Codes are exact (rint of the exact quotient, ties to even) and the integer sums
too, so what is left is float32: the sum's conversion, two scales and the bias,
2^-24 each of the values they round, then one rounding to the output's type.
"""
import pytest
import torch

DEV = "cuda"


@pytest.fixture(autouse=True, params=["native", "ctypes"])
def host_path(request, monkeypatch):
    """Every test on the native host path and on the Python one behind it."""
    if request.param == "ctypes":
        from quant_models import _native

        monkeypatch.setattr(_native, "host", lambda: None)


DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _codes(x):
    """(codes, scale) of the rows, from the definition."""
    xd = x.double()
    top = xd.abs().amax(-1, keepdim=True)
    q = torch.round(127 * xd / torch.where(top > 0, top, 1.0))  # exact where the quotient is a tie
    return q, (top[..., 0] / 127).float()  # in 64 bits: torch divides float32 by a number as a product on the device


def _check(y, x, w, sw, b):
    q, sx = _codes(x)
    prod = (q.reshape(-1, q.shape[-1]) @ w.double().t()) * sx.double().reshape(-1, 1) * sw.double()
    want = prod if b is None else prod + b.double()
    size = prod.abs() + (0 if b is None else b.double().abs())
    err = (y.double().reshape(want.shape) - want).abs()
    bound = HALF[y.dtype] * want.abs() + 4 * 2.0 ** -24 * (1 + HALF[y.dtype]) * size + 2.0 ** -25
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 768), (3, 7), (5, 515), (64, 64), (197, 768), (33, 4096), (2, 5000), (7, 4104)])
def test_codes_are_the_nearest(rows, k, dtype):
    from quant_models import ops

    g = _gen(rows * 10007 + k)
    x = (torch.randn(rows, k, device=DEV, generator=g) * torch.logspace(-6, 4, rows, device=DEV)[:, None]).to(dtype)
    if k > 4:  # exact ties: halves of the largest, and a row of zeros
        x[0, :5] = torch.tensor([2.0, 1.0, -1.0, 0.5, -2.0], device=DEV).to(dtype)
        x[0, 5:] = x[0, 5:].clamp(-2, 2)
        x[-1] = 0 if rows > 2 else x[-1]
    codes, scale = ops.quantize_int8(x)
    want, sw = _codes(x)
    assert codes.shape == x.shape and scale.shape == (rows,)
    assert torch.equal(codes.double(), want)
    assert torch.equal(scale, sw)


@pytest.mark.gpu
def test_codes_of_extreme_rows():
    """Subnormal and huge rows keep exact codes; inf and NaN make their row NaN."""
    from quant_models import ops

    base = torch.linspace(-1, 1, 64, device=DEV)
    rows = torch.stack([base * s for s in (1e-44, 1e-40, 2.0 ** -126, 1e-30, 3e38, 1e30)])
    codes, scale = ops.quantize_int8(rows)
    want, sw = _codes(rows)
    assert torch.equal(codes.double(), want) and torch.equal(scale, sw)
    for bad in (float("inf"), -float("inf"), float("nan")):
        x = base.repeat(3, 1)
        x[1, 5] = bad
        codes, scale = ops.quantize_int8(x)
        assert bool(torch.isnan(scale[1])) and bool((codes[1] == 0).all()) and bool(torch.isfinite(scale[[0, 2]]).all())
        w, ws = ops.quantize_int8(torch.randn(40, 64, device=DEV, generator=_gen(1)))
        y = ops.linear_int8(x, w, ws)
        assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[[0, 2]]).all())


SHAPES = [(1, 1, 1), (1, 768, 1000), (2, 16, 3), (8, 1024, 333), (16, 515, 64), (17, 768, 257), (31, 64, 31), (32, 80, 256),
          (33, 48, 255), (64, 130, 500), (65, 1024, 4), (129, 768, 1000), (300, 4096, 72), (777, 515, 333), (1576, 768, 2304),
          (3, 20000, 40), (40, 9000, 17), (16, 2048, 100), (2, 16384, 33), (1, 32768, 20), (5, 48, 17), (16, 2064, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_linear_int8_matches_its_definition(rows, k, n, dtype):
    from quant_models import ops

    g = _gen(rows + 31 * k + 1009 * n)
    x = torch.randn(rows, k, device=DEV, generator=g).to(dtype)
    w, sw = ops.quantize_int8(torch.randn(n, k, device=DEV, generator=g) * 0.02)
    b = torch.randn(n, device=DEV, generator=g) if rows % 2 else None
    y = ops.linear_int8(x, w, sw, b)
    assert y.shape == (rows, n) and y.dtype == dtype
    _check(y, x, w, sw, b)


@pytest.mark.gpu
def test_linear_int8_extreme_codes_sum_exactly():
    """Sums of K = 131072 products of 127 x 127 fill int32 and stay exact."""
    from quant_models import ops

    k = 131072
    x = torch.ones(3, k, device=DEV)
    x[1] = -1
    x[2, ::2] = -1
    w = torch.full((5, k), 127, dtype=torch.int8, device=DEV)
    y = ops.linear_int8(x, w, torch.ones(5, device=DEV))
    # the sum converted to float32, times float32(1 / 127): two roundings and that of the scale
    want = torch.tensor([127.0 * k, -127.0 * k, 0.0], device=DEV, dtype=torch.float64)[:, None]
    assert bool(((y.double() - want).abs() <= 3.01 * 2.0 ** -24 * want.abs()).all())


@pytest.mark.gpu
def test_linear_int8_takes_codes_strides_and_types():
    """Given codes, padded weight rows, leading dimensions, unaligned views,
    other output types and bias types: the same product."""
    from quant_models import ops

    g = _gen(5)
    x = torch.randn(3, 11, 100, device=DEV, generator=g).half()
    w, sw = ops.quantize_int8(torch.randn(70, 100, device=DEV, generator=g))
    b = torch.randn(70, device=DEV, generator=g)
    y = ops.linear_int8(x, w, sw, b)
    _check(y, x, w, sw, b)
    wide = torch.full((70, 128), 99, dtype=torch.int8, device=DEV)
    wide[:, :100] = w
    assert torch.equal(ops.linear_int8(x, wide[:, :100], sw, b), y)
    assert torch.equal(ops.linear_int8(x, w.t().contiguous().t(), sw, b), y)
    codes, sx = ops.quantize_int8(x)
    assert torch.equal(ops.linear_int8(codes, w, sw, b, out_dtype=torch.float16, x_scale=sx), y)
    assert torch.equal(ops.linear_int8(x, w, sw, b.double()), y)
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)
    flat[1:] = x.reshape(-1)
    assert torch.equal(ops.linear_int8(flat[1:].view(x.shape), w, sw, b), y)
    assert torch.equal(ops.linear_int8(x.transpose(0, 1), w, sw, b), y.transpose(0, 1))
    y32 = ops.linear_int8(x, w, sw, b, out_dtype=torch.float32)
    assert y32.dtype == torch.float32 and torch.equal(y32.half(), y)
    x64, w64 = torch.randn(40, 64, device=DEV, generator=g), torch.randint(-127, 128, (24, 64), device=DEV, dtype=torch.int8)
    s64 = torch.rand(24, device=DEV)
    want = ops.linear_int8(x64, w64, s64)
    off = torch.empty(24 * 64 + 8, dtype=torch.int8, device=DEV)
    off[8:] = w64.reshape(-1)
    assert torch.equal(ops.linear_int8(x64, off[8:].view(24, 64), s64), want)
    c64, sx = ops.quantize_int8(x64)
    off = torch.empty(40 * 64 + 3, dtype=torch.int8, device=DEV)
    off[3:] = c64.reshape(-1)
    assert torch.equal(ops.linear_int8(off[3:].view(40, 64), w64, s64, out_dtype=torch.float32, x_scale=sx), want)
    for shape in ((0, 64), (3, 0, 64)):
        assert ops.linear_int8(torch.empty(shape, device=DEV), w64, s64).shape == shape[:-1] + (24,)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 8, 300])
def test_linear_int8_on_streams_and_in_graphs(rows):
    from quant_models import ops

    g = _gen(rows)
    w, sw = ops.quantize_int8(torch.randn(500, 768, device=DEV, generator=g))
    x = torch.randn(rows, 768, device=DEV, generator=g).half()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.linear_int8(x, w, sw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ops.linear_int8(x, w, sw))
    static = x.clone()
    graphs = []
    for _ in range(2):
        ops.linear_int8(static, w, sw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear_int8(static, w, sw)
        graphs.append((graph, out))
    for i in range(3):
        static.copy_(torch.randn(rows, 768, device=DEV, generator=g).half())
        for graph, out in graphs:
            graph.replay()
            want = ops.linear_int8(static, w, sw)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.gpu
def test_linear_int8_refusals():
    from quant_models import ops

    x, w, s = torch.randn(4, 32, device=DEV), torch.zeros(8, 32, dtype=torch.int8, device=DEV), torch.ones(8, device=DEV)
    for call in (lambda: ops.linear_int8(x, w.float(), s), lambda: ops.linear_int8(x[:, :16], w, s),
                 lambda: ops.linear_int8(x, w, s[:4]), lambda: ops.linear_int8(x, w, s.half()),
                 lambda: ops.linear_int8(x, w, s, torch.ones(3, device=DEV)), lambda: ops.linear_int8(x.cpu(), w, s),
                 lambda: ops.linear_int8(x, w, s.cpu()), lambda: ops.linear_int8(w[:4], w, s),
                 lambda: ops.linear_int8(x, w, s, x_scale=torch.ones(4, device=DEV)),
                 lambda: ops.quantize_int8(torch.empty(3, 0, device=DEV))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.linear_int8(x.double(), w, s)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.linear_int8(x.requires_grad_(), w, s)
    with pytest.raises(RuntimeError, match="131072"):
        ops.linear_int8(torch.zeros(1, 131088, device=DEV), torch.zeros(1, 131088, dtype=torch.int8, device=DEV), s[:1])


@pytest.mark.gpu
def test_codes_of_more_rows_than_a_launch_has_waves():
    """2^24 and a few rows: the waves take more than one each."""
    from quant_models import ops

    rows = (1 << 24) + 5
    x = torch.randn(rows, 8, device=DEV, generator=_gen(9), dtype=torch.float16)
    codes, scale = ops.quantize_int8(x)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        c, s = ops.quantize_int8(x[part].contiguous())
        assert torch.equal(codes[part], c) and torch.equal(scale[part], s)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """An output and an input of 4.6 GB: rows in the middle and at the end are
    the bits of calls on those rows alone."""
    from quant_models import ops

    rows, n = 70001, 32768
    x = torch.randn(rows, 64, device=DEV, generator=_gen(1), dtype=torch.float16)
    w, sw = ops.quantize_int8(torch.randn(n, 64, device=DEV, generator=_gen(2)))
    parts = (slice(0, 40), slice(32700, 33000), slice(65400, 65700), slice(rows - 300, rows))
    y = ops.linear_int8(x, w, sw)
    for part in parts:
        assert torch.equal(y[part], ops.linear_int8(x[part], w, sw))
    codes, scale = ops.quantize_int8(y)
    for part in parts:
        c, s = ops.quantize_int8(y[part])
        assert torch.equal(codes[part], c) and torch.equal(scale[part], s)
