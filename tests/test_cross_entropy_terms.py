"""Gradients of linear_cross_entropy beside 16-bit operands: as near to the
formula as float32 sums are.

Bounds as in test_linear_cross_entropy, but for dz: its two 16-bit terms lose
at most 2^-8 of 2^-8 of it (bf16) or 2^-11 of 2^-11 (fp16), and the products of
the second term take part in the same float32 sums (twice as many terms).
"""
import pytest
import test_linear_cross_entropy as base
import torch

DEV = "cuda"
TERMS = {torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}
host_path = base.host_path


# small D, where a logit's own bound stays below a single term's rounding; 128
# rows and more columns than one tile, all forms of the tile product
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,v,d", [(1, 300, 16), (5, 1000, 8), (64, 1000, 24), (130, 513, 33), (700, 2000, 16), (3000, 40, 16)])
def test_gradients_to_the_last_bits(m, v, d, dtype, monkeypatch):
    # twice float32's sums: 2 v 2^-24 of the magnitudes, for which _check allows v 2^-24
    monkeypatch.setitem(base.ROUND, dtype, TERMS[dtype] + max(m, v) * 2.0 ** -24)
    for smooth, reduction in ((0.0, "mean"), (0.1, "sum")):
        x, w, t, b = base._inputs(m, v, d, dtype, bias=True, ignored=0.2 if m > 3 else 0.0)
        base._check(x, w, t, b, smooth, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_error_of_a_batch_is_that_of_its_rounding(dtype):
    """The 2-norm of the gradients' error against 64 bits: the rounding of the
    result is half a step at most, whose mean square over values spread evenly
    in a binade is below (2^-8 / 1.7)^2 of them (bf16); one 16-bit term of dz put
    as much again to it."""
    from quant_models import ops

    m, v, d = 64, 1000, 768
    x, w, t, b = base._inputs(m, v, d, dtype, bias=True)
    leaves = [p.clone().requires_grad_() for p in (x, w, b)]
    got = torch.autograd.grad(ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], label_smoothing=0.1) * 1024.0, leaves)
    exact = [p.double().requires_grad_() for p in (x, w, b)]
    loss = torch.nn.functional.cross_entropy(exact[0] @ exact[1].t() + exact[2], t, label_smoothing=0.1) * 1024.0
    for g, e in zip(got, torch.autograd.grad(loss, exact)):
        rounded = float((e.to(dtype).double() - e).norm())
        # as the result's own rounding: the rest is 2^-16 (2^-22) of dz, 2^-4 of a step, and the sums' 2^-20
        assert float((g.double() - e).norm()) <= 1.1 * rounded


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [40, 400])
def test_rows_beside_an_infinite_upstream_gradient(m, dtype, bad):
    """grad_x of the finite rows is what it is without the other row (whose
    gradient, here 0 instead, takes no part in theirs), and finite."""
    from quant_models import ops

    x, w, t, b = base._inputs(m, 300, 64, dtype, True, 0.2)
    t[3] = 7
    g = torch.linspace(-900, 900, m, device=DEV)
    with_bad, without = g.clone(), g.clone()
    with_bad[3], without[3] = bad, 0.0

    def run(up):
        leaves = [p.clone().requires_grad_() for p in (x, w, b)]
        return torch.autograd.grad(ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="none"), leaves, up)

    got, want = run(with_bad), run(without)
    rows = torch.arange(m, device=DEV) != 3
    assert bool(torch.isfinite(got[0][rows]).all()) and torch.equal(got[0][rows], want[0][rows])
    assert not bool(torch.isfinite(got[0][3]).any()) and not bool(torch.isfinite(got[1][7]).any())
    base._check(x, w, t, b, 0.0, "none", without)
    # a row without a label keeps its gradient to itself, whatever it is
    t[3] = -100
    assert all(torch.equal(a, e) for a, e in zip(run(with_bad), run(without)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,v,d", [(60, 5000, 64), (60, 301, 61), (400, 5000, 64), (400, 301, 61)])
def test_rows_far_below_the_largest_upstream_gradient(m, v, d, dtype):
    """grad_x of rows 2^-25 of the largest's gradient is as exact as theirs."""
    from quant_models import ops

    x, w, t, b = base._inputs(m, v, d, dtype, True, 0.1)
    up = torch.logspace(16, -9, m, base=2.0, device=DEV)
    xs = x.clone().requires_grad_()
    (got,) = torch.autograd.grad(ops.linear_cross_entropy(xs, w, t, b, reduction="none"), xs, up)
    xd, wd = x.double(), w.double()
    z = xd @ wd.t() + b.double()
    p = torch.softmax(z, 1)
    q = torch.zeros_like(p)
    valid = t != -100
    q[valid, t[valid]] = 1.0
    dz = torch.where(valid, up.double(), 0.0)[:, None] * (p - q)
    zerr = (d + 2) * 2.0 ** -24 * (xd.abs() @ wd.abs().t() + b.double().abs()).amax(1)
    # p's own error, dz's two bf16 terms (2^-16; fp16: and the second terms' product,
    # 2^-8 of dz times 2^-8 of w), float32 sums of up to six products a class
    perr = torch.where(valid, up.double(), 0.0)[:, None] * p * (3 * zerr + 2.0 ** -20 * 10)[:, None]
    size = perr + dz.abs() * ({torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -15, torch.float32: 2.0 ** -22}[dtype] + 6 * v * 2.0 ** -24)
    want = dz @ wd
    # fp16's own steps end at 2^-24
    bound = base.HALF[dtype] * want.abs() + 1.01 * size @ wd.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (off / bound).amax(1)
