"""rms_norm, rms_norm_int8 and their gradients against the definition in 64 bits.

float32 arithmetic: a row's sum of squares is at most 64 + 8 additions deep (all
of one sign), so 1 / rms is within (73 / 2 + 4) 2^-24 of itself and y within 44
2^-24, before its one rounding to the type.  Codes are exact.
"""
import pytest
import torch

DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24
TINY = 2.0 ** -25  # half of fp16's smallest number
SHAPES = [(1, 1), (1, 768), (3, 7), (5, 515), (197, 768), (33, 1024), (7, 1025), (9, 2048), (4, 2056), (2, 4096), (3, 5001),
          (2, 8192), (2, 8200), (1, 16384), (777, 515), (4100, 64)]


@pytest.fixture(params=["native", "ctypes"])
def host_path(request, monkeypatch):
    if request.param == "ctypes":
        from quant_models import _native

        monkeypatch.setattr(_native, "host", lambda: None)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inputs(m, c, dtype, wdt, seed=0):
    g = _gen(seed + 31 * m + c)
    loud = 1 + 6 * (torch.rand(c, generator=g, device=DEV) < 0.05)
    x = (torch.randn(m, c, generator=g, device=DEV) * loud).to(dtype)
    r = torch.randn(m, c, generator=g, device=DEV).to(dtype)
    w = None if wdt is None else (1 + 0.3 * torch.randn(c, generator=g, device=DEV)).to(wdt)
    return x, r, w


def _norm(h, w, eps):
    hd = h.double()
    rstd = 1 / (hd.square().mean(-1, keepdim=True) + eps).sqrt()
    n = hd * rstd
    return (n if w is None else n * w.double()), n, rstd


def _check(got, want, slack=44):
    err = (got.double() - want).abs()
    bound = HALF[got.dtype] * want.abs() + slack * U * want.abs() * (1 + HALF[got.dtype]) + TINY
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,c", SHAPES)
def test_norm_matches_its_definition(m, c, dtype, host_path):
    from quant_models import ops

    for wdt in (None, torch.float32, dtype):
        x, r, w = _inputs(m, c, dtype, wdt)
        y = ops.rms_norm(x, w, 1e-5)
        assert y.dtype == dtype and y.shape == x.shape
        _check(y, _norm(x, w, 1e-5)[0])
        y, h = ops.rms_norm(x, w, 1e-5, residual=r)
        assert torch.equal(h, x + r)  # one float32 addition, rounded: torch's too
        _check(y, _norm(h, w, 1e-5)[0])


def _codes(h, w, eps):
    p = h.double() if w is None else h.double() * w.double()
    top = p.abs().amax(-1, keepdim=True)
    q = torch.round(127 * p / torch.where(top > 0, top, 1.0))
    return q, (top * _norm(h, None, eps)[2] / 127)[..., 0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,c", SHAPES)
def test_codes_are_the_nearest(m, c, dtype, host_path):
    from quant_models import ops

    for wdt in (None, torch.float32, dtype):
        x, r, w = _inputs(m, c, dtype, wdt, 5)
        if c > 8 and wdt is None:  # exact ties: halves of the largest
            x[0, :5] = torch.tensor([8.0, 4.0, -4.0, 2.0, -8.0], device=DEV).to(dtype)
            x[0, 5:] = x[0, 5:].clamp(-8, 8)
        for res in (None, r):
            codes, scale, *h = ops.rms_norm_int8(x, w, 1e-5, residual=res)
            hh = x if res is None else h[0]
            if res is not None:
                assert torch.equal(hh, x + r)
            want, sw = _codes(hh, w, 1e-5)
            assert codes.dtype == torch.int8 and scale.shape == (m,)
            assert torch.equal(codes.double(), want)
            assert bool(((scale.double() - sw).abs() <= 50 * U * sw).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [64, 3000])
def test_extreme_rows(dtype, c, host_path):
    """Squares past float32's range, rows of zeros, inf and NaN."""
    from quant_models import ops

    base = torch.linspace(-1, 1, c, device=DEV)
    x = torch.stack([base * s for s in (1e30, 3e38, 1e-30, 1.0, 0.0)]).to(dtype)
    y = ops.rms_norm(x, None, 1e-37)
    _check(y, _norm(x, None, 1e-37)[0])
    codes, scale = ops.rms_norm_int8(x, None, 1e-37)
    want, sw = _codes(x, None, 1e-37)
    assert torch.equal(codes.double(), want)
    assert bool(((scale.double() - sw).abs() <= 50 * U * sw).all()) and float(scale[4]) == 0
    for bad in (float("inf"), float("nan")):
        z = x.clone()
        z[3, 5] = bad
        codes, scale = ops.rms_norm_int8(z, None, 1e-6)
        assert bool(torch.isnan(scale[3])) and bool((codes[3] == 0).all()) and bool(torch.isfinite(scale[[0, 1, 2, 4]]).all())
        y = ops.rms_norm(z, None, 1e-6)
        assert bool(torch.isnan(y[3, 5])) and bool(torch.isfinite(y[[0, 2, 4]]).all())


def _grad_bounds(h, w, gy, gh, eps):
    """The formula's gradients and bounds of float32's own error."""
    _, n, rstd = _norm(h, None, eps)
    g = gy.double() if w is None else gy.double() * w.double()
    mean = (g * n).mean(-1, keepdim=True)
    size = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    gx = rstd * (g - n * mean)
    extra = 0
    if gh is not None:
        gx, extra = gx + gh.double(), gh.double().abs()
    gw, gw_size = (gy.double() * n).sum(0), (gy.double() * n).abs().sum(0)
    # n: 44 roundings, the mean of g n: 73 of its own and n's, four products
    return gx, 200 * U * size + 2 * U * extra, gw, (h.shape[0] + 200) * U * gw_size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,c", SHAPES)
def test_gradients_match_the_formula(m, c, dtype):
    from quant_models import ops

    for wdt, with_res, both in ((torch.float32, True, True), (dtype, True, False), (None, False, False), (dtype, False, False)):
        x, r, w = _inputs(m, c, dtype, wdt, 9)
        g = _gen(m + c)
        gy, gh = (torch.randn(m, c, generator=g, device=DEV).to(dtype) for _ in range(2))
        leaves = [t.requires_grad_() for t in ([x, r] if with_res else [x]) + ([w] if w is not None else [])]
        out = ops.rms_norm(x, w, 1e-6, residual=r if with_res else None)
        y, h = out if with_res else (out, x)
        grads = torch.autograd.grad([y, h] if both else [y], leaves, [gy, gh] if both else [gy])
        gx, bx, gw, bw = _grad_bounds(h.detach(), w, gy, gh if both else None, 1e-6)
        for got in grads[:2] if with_res else grads[:1]:
            err = (got.double() - gx).abs()
            assert bool((err <= bx * (1 + HALF[dtype]) + HALF[dtype] * gx.abs() + TINY).all()), float(err.max())
        if w is not None:
            err = (grads[-1].double() - gw).abs()
            assert bool((err <= bw * (1 + HALF[wdt]) + HALF[wdt] * gw.abs() + TINY).all()), float(err.max())


@pytest.mark.gpu
def test_gradients_match_differences():
    """Against central differences of the definition in 64 bits: steps of 1e-5
    leave 1e-10 of the third derivative and 1e-11 of rounding, float32 2e-5."""
    from quant_models import ops

    g = _gen(3)
    x, r, w = (torch.randn(*s, generator=g, device=DEV) for s in ((6, 40), (6, 40), (40,)))
    gy, gh = (torch.randn(6, 40, generator=g, device=DEV) for _ in range(2))
    y, h = ops.rms_norm(x.requires_grad_(), w.requires_grad_(), 1e-3, residual=r.requires_grad_())
    grads = torch.autograd.grad([y, h], [x, r, w], [gy, gh])

    def f(x, r, w):
        hd = x + r
        return ((hd / (hd.square().mean(-1, keepdim=True) + 1e-3).sqrt() * w) * gy.double()).sum() + (hd * gh.double()).sum()

    at = [t.detach().double() for t in (x, r, w)]
    for i in range(3):
        d = torch.randn(at[i].shape, generator=g, device=DEV, dtype=torch.float64)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-5 * d, at[i] - 1e-5 * d
        want = (f(*up) - f(*down)) / 2e-5
        got = (grads[i].double() * d).sum()
        assert abs(float(got - want)) <= 200 * U * float((grads[i].double() * d).abs().sum()) * 10 + 1e-6


@pytest.mark.gpu
def test_layouts_streams_and_unused_outputs():
    from quant_models import ops

    x, r, w = _inputs(40, 768, torch.bfloat16, torch.float32)
    want, hw = ops.rms_norm(x, w, 1e-6, residual=r)
    wide = torch.cat([x, x], 1)
    for form in (x.t().contiguous().t(), wide[:, 768:], torch.zeros(40 * 768 + 1, device=DEV, dtype=x.dtype)[1:].view(40, 768).copy_(x)):
        y, h = ops.rms_norm(form, w, 1e-6, residual=r)
        assert torch.equal(y, want) and torch.equal(h, hw)
        assert all(torch.equal(a, b) for a, b in zip(ops.rms_norm_int8(form, w, residual=r), ops.rms_norm_int8(x, w, residual=r)))
    y, h = ops.rms_norm(x.view(4, 10, 768), w, 1e-6, residual=r.view(4, 10, 768))
    assert y.shape == (4, 10, 768) and torch.equal(y.view(40, 768), want)
    codes, scale = ops.rms_norm_int8(x.view(4, 10, 768), w)
    assert codes.shape == (4, 10, 768) and scale.shape == (4, 10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.rms_norm(x, w, 1e-6, residual=r)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    assert ops.rms_norm(x[:0], w).shape == (0, 768)
    assert ops.rms_norm_int8(x[:0], w)[1].shape == (0,)
    # only the sum is used, only the weight is trained, a gradient that is not contiguous
    xg, rg, wg = x.clone().requires_grad_(), r.clone().requires_grad_(), w.clone().requires_grad_()
    y, h = ops.rms_norm(xg, wg, 1e-6, residual=rg)
    h.float().sum().backward()
    assert bool((xg.grad == 1).all()) and bool((rg.grad == 1).all()) and wg.grad is None
    (gw,) = torch.autograd.grad(ops.rms_norm(x, wg, 1e-6), wg, torch.ones(768, 40, device=DEV, dtype=x.dtype).t())
    assert torch.equal(gw, torch.autograd.grad(ops.rms_norm(x, wg, 1e-6), wg, torch.ones_like(x))[0])


@pytest.mark.gpu
def test_twice_differentiated_is_refused():
    from quant_models import ops

    x = torch.randn(3, 8, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(ops.rms_norm(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()


@pytest.mark.gpu
def test_captured_training_step_replays():
    from quant_models import ops

    x, r, w = _inputs(50, 515, torch.float32, torch.float32)
    leaves = [t.requires_grad_() for t in (x, r, w)]

    def step():
        y, h = ops.rms_norm(x, w, 1e-6, residual=r)
        return torch.autograd.grad(y.square().sum() + h.sum(), leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        ops.rms_norm(x.detach(), w.detach())  # eager work between the replays
    torch.cuda.synchronize()
    with torch.enable_grad():
        alive = ops.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(ops.rms_norm(x, w).sum(), leaves[:1])
    alive.sum().backward()


@pytest.mark.gpu
def test_refusals():
    from quant_models import ops

    x, r, w = _inputs(4, 16, torch.float32, torch.float32)
    for bad in (lambda: ops.rms_norm(x.cpu()), lambda: ops.rms_norm(x, w[:8]), lambda: ops.rms_norm(x, w, 0.0), lambda: ops.rms_norm(x, w, float("nan")),
                lambda: ops.rms_norm(x, w, residual=r[:2]), lambda: ops.rms_norm(x, w, residual=r.half()), lambda: ops.rms_norm(x[0, 0]),
                lambda: ops.rms_norm(x, w.cpu()), lambda: ops.rms_norm(torch.zeros(1, 16385, device=DEV)), lambda: ops.rms_norm_int8(x, w, -1.0)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.rms_norm(x.double()), lambda: ops.rms_norm(x, w.double()), lambda: ops.rms_norm_int8(x.long())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.rms_norm_int8(x.requires_grad_(), w)


@pytest.mark.gpu
def test_gradients_without_the_native_path_are_refused(monkeypatch):
    from quant_models import _native, ops

    monkeypatch.setattr(_native, "host", lambda: None)
    with pytest.raises(RuntimeError, match="native host path"):
        ops.rms_norm(torch.randn(2, 8, device=DEV, requires_grad=True))


def test_argument_errors():
    from quant_models import _native as N

    L, at = N.load(), 1 << 20  # an aligned address that is never dereferenced

    def norm(x=at, r=None, dt=1, m=4, c=32, w=at, wdt=0, eps=1e-6, y=at, h=None, stat=None):
        return L.rpfq_rms_norm(x, r, dt, m, c, w, wdt, eps, y, h, stat, None)

    def codes(x=at, r=None, dt=1, m=4, c=32, w=at, wdt=0, eps=1e-6, q=at, s=at, h=None):
        return L.rpfq_rms_norm_int8(x, r, dt, m, c, w, wdt, eps, q, s, h, None)

    def grad(gy=at, gh=None, h=at, dt=1, m=4, c=32, w=at, wdt=0, stat=at, gx=at, gw=at, work=at, nb=1 << 30):
        return L.rpfq_rms_norm_grad(gy, gh, h, dt, m, c, w, wdt, stat, gx, gw, work, nb, None)

    assert norm(x=None) == 1 and norm(y=None) == 1 and norm(r=at) == 1 and norm(h=at) == 1
    assert codes(x=None) == 1 and codes(q=None) == 1 and codes(s=None) == 1 and codes(r=at) == 1
    assert grad(gy=None) == 1 and grad(h=None) == 1 and grad(stat=None) == 1 and grad(gx=None) == 1 and grad(work=None) == 1
    assert grad(w=None) == 1
    for f in (norm, codes, grad):
        assert f(dt=3) == 5 and f(wdt=-1) == 5 and f(m=0) == 2 and f(c=0) == 2 and f(c=16385) == 2 and f(m=(1 << 30) + 1) == 2
    for f in (norm, codes):
        assert f(eps=0.0) == 6 and f(eps=float("nan")) == 6 and f(eps=float("inf")) == 6 and f(x=at + 1) == 3 and f(w=at + 2) == 3
    assert grad(nb=0) == 2 and grad(work=at + 16) == 3 and grad(gx=at + 1) == 3
    assert L.rpfq_rms_norm_grad_workspace_bytes(0, 5) == 0 and L.rpfq_rms_norm_grad_workspace_bytes(4, 32) >= 128
