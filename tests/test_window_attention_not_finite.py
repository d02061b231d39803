"""Values that are not finite in window_attention and its form over a cache, where
rows are joined from parts and where a sequence ends: they reach what sees them,
all of it, and nothing else."""
import math

import pytest
import torch

import test_window_attention as W

DEV = W.DEV


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_gradients_behind_the_end_of_divided_sinks(which, causal, dtype):
    """Sinks whose far ranges are divided among workgroups, and a sequence that ends
    among them: zeros behind its end, though its own values are not finite."""
    from quant_models import ops

    q, k, v, go = W._inputs(2, 900, 4, 1, 32, dtype, 3)
    (q, k, v)[which][1, 5, 0, 0] = math.inf
    lens = torch.tensor([900, 20], dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.window_attention(*leaves, 9, 65, causal=causal, lengths=lens)
    assert not bool(out[1, 20:].any())
    for grad in torch.autograd.grad(out, leaves, go):
        assert bool(grad[0].isfinite().all())
        assert not bool(grad[1, 20:].any())  # any() of NaN is true
