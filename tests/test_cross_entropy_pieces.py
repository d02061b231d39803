"""Classes whose logits' gradient does not fit one piece of 1 GiB (2 bytes a
term, two terms beside 16-bit operands, three beside float32): what the second
piece takes from the first and from its own place, biases, rows without a
label, smoothing, all gradients.  Bounds as in test_linear_cross_entropy."""
import pytest
import test_linear_cross_entropy as base
import torch

M, V = 20011, 14003


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,reduction", [(16, "sum"), (17, "mean"), (16, "none")])
def test_gradients_over_two_pieces(dtype, d, reduction):
    x, w, t, b = base._inputs(M, V, d, dtype, bias=True, ignored=0.3)
    t[:4] = torch.tensor([0, V - 1, V // 2, 7168], device=base.DEV)  # 7168: where the second piece begins
    # 16-bit gradients of a mean stay normal numbers
    up = {"sum": None, "mean": torch.tensor(8192.0, device=base.DEV), "none": torch.linspace(-2, 2, M, device=base.DEV)}[reduction]
    base._check(x, w, t, b, 0.1, reduction, up)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_that_hold_anything_over_two_pieces(dtype):
    """The copy of x without its ignored rows serves both pieces."""
    from quant_models import ops

    x, w, t, b = base._inputs(M, V, 16, dtype, bias=True, ignored=0.3)
    dirty = x.clone()
    dirty[t == -100] = float("nan")

    def run(x):
        leaves = [p.clone().requires_grad_() for p in (x, w, b)]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        return (loss.detach(),) + torch.autograd.grad(loss, leaves, torch.tensor(8192.0, device=base.DEV))

    for a, e in zip(run(dirty), run(x)):
        assert torch.equal(a, e)
