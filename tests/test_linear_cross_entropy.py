"""linear_cross_entropy and its gradients against the formula in 64 bits.

Bounds.  A logit is a float32 sum of D products: off by at most (D + 2) 2^-24
of sum |x| |w| + |b|.  exp and log in float32 add 2^-20 (1 + ln V + |lse|).
dz is p - q, relative error of p from the two above, rounded once to 16 bits
(2^-8 bf16, 2^-11 fp16; nothing for float32), and the gradients' sums of n
terms add n 2^-24 of the sum of magnitudes, then one rounding to their type.
"""
import math

import pytest
import torch
import torch.nn.functional as F

DEV = "cuda"


@pytest.fixture(autouse=True, params=["native", "ctypes"])
def host_path(request, monkeypatch):
    """Every test on the native host path and on the Python one behind it."""
    if request.param == "ctypes":
        from quant_models import _native

        monkeypatch.setattr(_native, "host", lambda: None)


HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ROUND = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # of dz


def _inputs(m, v, d, dtype, bias, ignored=0.0, seed=0, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed + m + 7 * v + 13 * d)
    w = torch.randn(v, d, device=DEV, generator=g) * (spread / math.sqrt(d))
    t = torch.randint(0, v, (m,), device=DEV, generator=g)
    x = torch.randn(m, d, device=DEV, generator=g) + 2 * (torch.rand(m, 1, device=DEV, generator=g) < 0.5) * w[t]
    b = torch.randn(v, device=DEV, generator=g) if bias else None
    t[torch.rand(m, device=DEV, generator=g) < ignored] = -100
    if m > 1:
        t[0], t[-1] = v - 1, 0
    return x.to(dtype), w.to(dtype), t, None if b is None else b.to(dtype)


def _check(x, w, t, b, smooth=0.0, reduction="mean", grad=None, ignore=-100):
    """One call and its gradients against 64 bits."""
    from quant_models import ops

    m, d = x.shape
    v = w.shape[0]
    xs, ws = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    bs = None if b is None else b.detach().clone().requires_grad_()
    loss = ops.linear_cross_entropy(xs, ws, t, bs, ignore_index=ignore, label_smoothing=smooth, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == ((m,) if reduction == "none" else ())
    up = torch.ones_like(loss) if grad is None else grad
    got = torch.autograd.grad(loss, [xs, ws] + ([bs] if bs is not None else []), up)
    xd, wd = x.double(), w.double()
    valid = t != ignore
    xd = torch.where(valid[:, None], xd, 0.0)
    z = xd @ wd.t() + (0 if b is None else b.double())
    zerr = (d + 2) * 2.0 ** -24 * (xd.abs() @ wd.abs().t() + (0 if b is None else torch.nan_to_num(b.double(), neginf=0).abs()))
    zerr = zerr.amax(1)
    lse = torch.logsumexp(z, 1)
    q = torch.full_like(z, smooth / v)
    q[valid, t[valid]] += 1 - smooth
    rows = torch.where(valid, -(torch.where(q > 0, q * torch.log_softmax(z, 1), 0.0)).sum(1), 0.0)
    rerr = torch.where(valid, 3 * zerr + 2.0 ** -20 * (1 + math.log(v) + lse.abs()), 0.0)
    count = valid.sum()
    if reduction == "none":
        want, lerr, gm = rows, rerr, up.double()
    elif reduction == "sum":
        want, lerr, gm = rows.sum(), rerr.sum(), up.double().expand(m)
    else:
        want, lerr, gm = rows.sum() / count, rerr.sum() / count, up.double().expand(m) / count
    err = (loss.double() - want).abs()
    assert bool((err <= lerr + 2.0 ** -22 * want.abs()).all()), (float(err.max()), float(lerr.max()))
    p = torch.softmax(z, 1)
    gm = torch.where(valid, gm, 0.0)
    dz = (p - q) * gm[:, None]
    # p's own error, then the rounding of dz
    u = HALF[x.dtype]
    perr = p * (3 * zerr + 2.0 ** -20 * (1 + math.log(v)))[:, None] * gm.abs()[:, None]
    zz = dz.abs() * ROUND[x.dtype] + perr + (2.0 ** -39 * gm.abs().max() if x.dtype == torch.float16 else 0)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -140
    for name, g, e, b1 in (("x", got[0], dz @ wd, zz @ wd.abs() + v * 2.0 ** -24 * (dz.abs() @ wd.abs())),
                           ("w", got[1], dz.t() @ xd, zz.t() @ xd.abs() + m * 2.0 ** -24 * (dz.abs().t() @ xd.abs()))):
        assert g.dtype == x.dtype
        bound = 1.01 * (u * e.abs() + (1 + u) * b1 + tiny) + 2.0 ** -22 * e.abs()
        off = (g.double() - e).abs()
        assert bool((off <= bound).all()), (name, float((off - bound).max()), float(off.max()))
    if b is not None:
        e = dz.sum(0)
        # db: float32 sums of the unrounded dz
        bound = 1.01 * (HALF[b.dtype] * e.abs() + 2 * perr.sum(0) + (m + 8) * 2.0 ** -24 * dz.abs().sum(0) + tiny)
        off = (got[2].double() - e).abs()
        assert got[2].dtype == b.dtype and bool((off <= bound).all()), ("b", float((off - bound).max()))
    return loss, got


SHAPES = [(1, 2, 1), (1, 1000, 768), (3, 7, 5), (2, 256, 64), (31, 257, 33), (33, 255, 96), (64, 1000, 768), (65, 513, 100),
          (128, 100, 385), (200, 5000, 192), (300, 3001, 384), (1000, 777, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,v,d", SHAPES)
def test_loss_and_gradients(m, v, d, dtype):
    x, w, t, b = _inputs(m, v, d, dtype, bias=(m + v) % 2 == 0, ignored=0.3 if m > 30 else 0.0)
    _check(x, w, t, b, smooth=0.1 if d % 2 else 0.0, reduction="mean" if m % 3 else "sum")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_with_gradients_of_their_own(dtype):
    """reduction none: gradients over many magnitudes, zeros among them."""
    x, w, t, b = _inputs(70, 300, 64, dtype, True, 0.2)
    g = torch.logspace(-3, 3, 70, device=DEV) * torch.where(torch.arange(70, device=DEV) % 2 == 0, 1.0, -1.0)
    g[5] = 0
    _check(x, w, t, b, 0.2, "none", g)
    _check(x, w, t, b, 0.0, "none", torch.zeros_like(g))


@pytest.mark.gpu
def test_gradients_against_differences():
    """float32 gradients against central differences of the 64-bit loss."""
    from quant_models import ops

    x, w, t, b = _inputs(6, 9, 8, torch.float32, True)
    leaves = [p.clone().requires_grad_() for p in (x, w, b)]
    grads = torch.autograd.grad(ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], label_smoothing=0.1), leaves)
    base = [p.double() for p in (x, w, b)]
    h = 1e-5
    for which, g in enumerate(grads):
        for i in range(0, base[which].numel(), 5):
            ends = []
            for s in (h, -h):
                p = [q.clone() for q in base]
                p[which].view(-1)[i] += s
                ends.append(float(F.cross_entropy(F.linear(p[0], p[1], p[2]), t, label_smoothing=0.1)))
            # differences: h^2 / 6 of a third derivative below 10^2, and 1e-16 / h
            assert abs((ends[0] - ends[1]) / (2 * h) - float(g.view(-1)[i])) <= 1e-7 + 2e-6 * float(g.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ignored_rows_may_hold_anything(dtype):
    """NaN and inf in rows without a label reach nothing; their grad_x is 0.
    All rows without one: loss NaN (mean) or 0 (sum), gradients 0."""
    from quant_models import ops

    x, w, t, b = _inputs(140, 300, 72, dtype, True, 0.4)
    dirty = x.clone()
    bad = torch.where(t == -100)[0]
    dirty[bad[0]], dirty[bad[1], 3], dirty[bad[2], 5] = float("nan"), float("inf"), -float("inf")
    loss, grads = _check(x, w, t, b, 0.1)
    leaves = [p.clone().requires_grad_() for p in (dirty, w, b)]
    again = ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], label_smoothing=0.1)
    assert torch.equal(again, loss)
    for a, e in zip(torch.autograd.grad(again, leaves), grads):
        assert torch.equal(a, e)
    assert bool((grads[0][bad] == 0).all())
    none = torch.full_like(t, -100)
    for reduction in ("mean", "sum"):
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], none, leaves[2], reduction=reduction)
        assert math.isnan(loss.item()) if reduction == "mean" else loss.item() == 0
        assert all(bool((g == 0).all()) for g in torch.autograd.grad(loss, leaves))


@pytest.mark.gpu
def test_masked_classes_and_special_values():
    """Classes masked by a bias of -inf or the type's lowest value, large
    logits, and NaN where torch has it."""
    from quant_models import ops

    for dtype in (torch.bfloat16, torch.float32):
        x, w, t, b = _inputs(40, 600, 64, dtype, True)
        for low in (-float("inf"), torch.finfo(dtype).min):
            bm = b.clone()
            bm[256:512] = low  # a whole tile of classes
            bm[3] = low
            tt = torch.where((t >= 256) & (t < 512) | (t == 3), 1, t)
            loss = ops.linear_cross_entropy(x, w, tt, bm, reduction="none")
            want = F.cross_entropy(F.linear(x.double(), w.double(), bm.double()), tt, reduction="none")
            assert bool(((loss.double() - want).abs() <= 2.0 ** -15 * (1 + want.abs())).all())
            leaves = [p.clone().requires_grad_() for p in (x, w, bm)]
            gx, gw, gb = torch.autograd.grad(ops.linear_cross_entropy(leaves[0], leaves[1], tt, leaves[2]), leaves)
            assert bool((gw[256:512] == 0).all()) and bool((gb[256:512] == 0).all()) and bool(torch.isfinite(gx).all())
            # a label whose class is masked: infinite loss
            tt[0] = 300
            if low == -float("inf"):
                assert float(ops.linear_cross_entropy(x, w, tt, bm, reduction="none")[0]) == float("inf")
    x, w, t, _ = _inputs(20, 300, 64, torch.float32, False)
    loss = ops.linear_cross_entropy(x * 1e3, w * 1e2, t, reduction="none")
    want = F.cross_entropy(F.linear((x * 1e3).double(), (w * 1e2).double()), t, reduction="none")
    assert bool(((loss.double() - want).abs() <= 2.0 ** -16 * want.abs().max()).all())
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[4, 2] = bad
        loss = ops.linear_cross_entropy(y, w, t, reduction="none")
        assert bool(torch.isnan(loss[4])) and bool(torch.isfinite(loss[torch.arange(20) != 4]).all())
    t[2], t[3] = 300, -1  # no classes
    loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    assert bool(torch.isnan(loss[2:4]).all()) and int(torch.isnan(loss).sum()) == 2


@pytest.mark.gpu
def test_pieces_and_splits_agree(monkeypatch):
    """Many rows against few classes (split over the rows) and the pieces of a
    large vocabulary: the formula's gradients."""
    x, w, t, b = _inputs(6000, 40, 64, torch.bfloat16, True, 0.1)
    _check(x, w, t, b)
    x, w, t, b = _inputs(40, 30000, 64, torch.float16, True, 0.1)
    _check(x, w, t, b)


@pytest.mark.gpu
def test_more_than_one_piece():
    """dz of 150,000 rows x 8,000 classes does not fit one piece: the gradients
    of the pieces join.  Against the formula in float32 on the same operands."""
    from quant_models import ops

    m, v, d = 150_000, 8_000, 16
    x, w, t, _ = _inputs(m, v, d, torch.bfloat16, False)
    leaves = [p.clone().requires_grad_() for p in (x, w)]
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t)
    gx, gw = torch.autograd.grad(loss, leaves)
    z = x.float() @ w.float().t()
    total = torch.logsumexp(z, 1)
    assert abs(float(loss) - float((total - z.gather(1, t[:, None])[:, 0]).double().mean())) <= 2.0 ** -16
    dz = z.sub_(total[:, None]).exp_()
    p = dz.clone()
    dz.scatter_add_(1, t[:, None], torch.full((m, 1), -1.0, device=DEV))
    # p in float32 is off by 2^-20 (1 + ln V) of itself on either side, which is
    # most of p - 1 where that is small (a label answered with p = 0.9999)
    off = 2 * 2.0 ** -20 * (1 + math.log(v)) * p
    for g, e, size in ((gx, dz @ w.float() / m, (dz.abs() * (2.0 ** -8 + 2.0 ** -10) + off) @ w.float().abs() / m),
                       (gw, dz.t() @ x.float() / m, (dz.abs() * (2.0 ** -8 + 2.0 ** -10) + off).t() @ x.float().abs() / m)):
        # dz's rounding and the gradient's, and float32 sums of up to 150,000 terms on both sides
        assert bool(((g.float() - e).abs() <= 2.0 ** -8 * e.abs() + size).all())


@pytest.mark.gpu
def test_same_bits_twice_other_stream_and_views():
    from quant_models import ops

    x, w, t, b = _inputs(333, 1001, 72, torch.bfloat16, True, 0.1)

    def call(x, w, t, b):
        leaves = [p.detach().requires_grad_() for p in (x, w, b)]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        return (loss.detach(),) + torch.autograd.grad(loss, leaves)

    first = call(x, w, t, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(x, w, t, b)
    torch.cuda.current_stream().wait_stream(side)
    wide = torch.randn(333, 200, device=DEV).bfloat16()
    wide[:, 5:77] = x
    off = torch.empty(1001 * 72 + 1, dtype=w.dtype, device=DEV)
    off[1:] = w.reshape(-1)
    views = call(wide[:, 5:77], off[1:].view(1001, 72), t, b)
    for a, c, e in zip(first, other, views):
        assert torch.equal(a, c) and torch.equal(a, e)
    shaped = ops.linear_cross_entropy(x[:330].view(3, 110, 72), w, t[:330].view(3, 110), b, reduction="none")
    assert torch.equal(shaped.view(-1), ops.linear_cross_entropy(x[:330], w, t[:330], b, reduction="none"))


@pytest.mark.gpu
def test_some_gradients_only_and_autocast():
    from quant_models import ops

    x, w, t, b = _inputs(90, 300, 64, torch.float32, True)
    xs = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(ops.linear_cross_entropy(xs, w, t, b), [xs])
    ws = w.clone().requires_grad_()
    (gw,) = torch.autograd.grad(ops.linear_cross_entropy(x, ws, t, b), [ws])
    bs = b.clone().requires_grad_()
    (gb,) = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, bs), [bs])
    leaves = [p.clone().requires_grad_() for p in (x, w, b)]
    for a, e in zip(torch.autograd.grad(ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2]), leaves), (gx, gw, gb)):
        assert torch.equal(a, e)
    assert not ops.linear_cross_entropy(x, w, t, b).requires_grad
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
    got = torch.autograd.grad(loss, leaves)
    low = [leaves[0].detach().bfloat16().requires_grad_(), leaves[1].detach().bfloat16().requires_grad_()]
    want = ops.linear_cross_entropy(low[0], low[1], t, b)
    assert torch.equal(loss, want) and got[0].dtype == torch.float32
    for a, e in zip(got, torch.autograd.grad(want, low)):
        assert torch.equal(a, e.float())


@pytest.mark.gpu
@pytest.mark.parametrize("m,v", [(48, 1000), (300, 3000)])
def test_captured_steps_replay(m, v):
    """Forward and backward in a graph, replayed on other operands."""
    from quant_models import ops

    x, w, t, b = _inputs(m, v, 64, torch.bfloat16, True, 0.1)
    leaves = [p.clone().requires_grad_() for p in (x, w, b)]

    def call():
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], label_smoothing=0.1)
        return (loss,) + torch.autograd.grad(loss, leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        x2, w2, t2, b2 = _inputs(m, v, 64, torch.bfloat16, True, 0.2, seed=100 + i)
        with torch.no_grad():
            for dst, src in zip(leaves + [t], (x2, w2, b2, t2)):
                dst.copy_(src)
        graph.replay()
        got = [o.detach().clone() for o in out]
        want = [o.detach() for o in call()]
        torch.cuda.synchronize()
        for a, e in zip(got, want):
            assert torch.equal(a, e)


@pytest.mark.gpu
def test_no_rows_and_refusals():
    from quant_models import ops

    x, w, t, b = _inputs(4, 10, 8, torch.float32, True)
    for reduction in ("none", "sum", "mean"):
        leaves = [p.requires_grad_() for p in (x[:0].clone(), w.clone(), b.clone())]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t[:0], leaves[2], reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ())
        assert reduction == "none" or math.isnan(float(loss)) == (reduction == "mean")
        grads = torch.autograd.grad(loss.sum(), leaves)
        assert all(g.shape == p.shape and bool((g == 0).all()) for g, p in zip(grads, leaves))
    for call in (lambda: ops.linear_cross_entropy(x.cpu(), w, t), lambda: ops.linear_cross_entropy(x, w.cpu(), t),
                 lambda: ops.linear_cross_entropy(x, w, t.cpu()), lambda: ops.linear_cross_entropy(x[:, :5], w, t),
                 lambda: ops.linear_cross_entropy(x, w, t.int()), lambda: ops.linear_cross_entropy(x, w, t[:2]),
                 lambda: ops.linear_cross_entropy(x, w, t, b[:3]), lambda: ops.linear_cross_entropy(x, w[:0], t),
                 lambda: ops.linear_cross_entropy(x, w, t, reduction="max"),
                 lambda: ops.linear_cross_entropy(x, w, t, label_smoothing=1.5)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.linear_cross_entropy(x.half(), w, t), lambda: ops.linear_cross_entropy(x.double(), w.double(), t),
                 lambda: ops.linear_cross_entropy(x, w, t, b.double())):
        with pytest.raises(TypeError):
            call()
    xs = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(ops.linear_cross_entropy(xs, w, t), [xs], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
def test_weights_of_more_than_4_gb():
    """1.2 M classes of 2,048 fp16 features; the gradient of some of the first,
    middle and last classes in 64 bits, times 2^12 to stay fp16 normals.  A
    logit is off by le = (D + 2) 2^-24 sum |x| |w|, p by twice that of itself
    and the exponentials' 2^-20 (1 + ln V + |lse|); dz is rounded to 2^-11."""
    from quant_models import ops

    m, v, d = 64, 1200000, 2048
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(m, d, device=DEV, generator=g, dtype=torch.float16).requires_grad_()
    w = (torch.randn(v, d, device=DEV, generator=g, dtype=torch.float16) / math.sqrt(d)).requires_grad_()
    t = torch.randint(0, v, (m,), device=DEV, generator=g)
    t[:3] = torch.tensor([v - 1, v - 200, 0], device=DEV)
    loss = ops.linear_cross_entropy(x, w, t, reduction="sum")
    loss.backward(torch.tensor(4096.0, device=DEV))
    xd = x.detach().double()
    lse = torch.stack([torch.logsumexp(xd @ c.detach().double().t(), 1) for c in w.split(50000)], 1).logsumexp(1)
    le = (d + 2) * 2.0 ** -24 * (xd.abs() @ w.detach()[:50000].abs().double().t()).max() * 1.5  # rows of w are alike
    zt = (xd * w.detach()[t].double()).sum(1)
    assert abs(float(loss.detach().double() - (lse - zt).sum())) <= m * float(2 * le + 2.0 ** -20 * (1 + math.log(v) + lse.max()))
    for part in (slice(0, 300), slice(524200, 524500), slice(1048500, 1048800), slice(v - 300, v)):
        c = torch.arange(v, device=DEV)[part]
        p = torch.exp(xd @ w.detach()[part].double().t() - lse[:, None])
        dz = p - (t[:, None] == c).double()
        off = p * (2 * le + 2.0 ** -20 * (1 + math.log(v) + lse.max())) + 2.0 ** -11 * dz.abs() + 2.0 ** -40
        want = 4096 * dz.t() @ xd
        bound = 2.0 ** -11 * want.abs() + 4096 * (off + m * 2.0 ** -24 * dz.abs()).t() @ xd.abs() + 2.0 ** -25
        assert bool(((w.grad[part].double() - want).abs() <= bound * (1 + 2.0 ** -10)).all()), part
