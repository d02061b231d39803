"""rotary over more tokens than one launch has workgroups for."""
import pytest
import torch

import test_rotary as R

DEV = R.DEV


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_tokens_past_a_launch(interleaved):
    """130 pairs: a token a workgroup, so 2^24 tokens would be a grid of 2^32 threads."""
    from quant_models import ops

    n, d, sections = (1 << 24) + 77, 262, (130,)
    g = R._gen(3)
    x = torch.randn(1, 1, 1, d, generator=g, device=DEV).half().expand(1, n, 1, d)
    positions, freqs = torch.arange(n, dtype=torch.int32, device=DEV), R._freqs(sections)
    out = ops.rotary(x, positions, freqs, sections, interleaved=interleaved)
    half = 1 << 23
    at = torch.tensor([0, 1, half - 1, half, half + 1, 2 * half - 1, 2 * half, n - 2, n - 1], device=DEV)
    R._check(out[:, at], *R._turned(x[:, at], positions[at][:, None], freqs, sections, interleaved))
    # no token was left: a turn keeps a head's length, and the values behind the pairs
    assert torch.equal(out[..., 260:], x[..., 260:])
    size = x[0, 0, 0].float().norm()
    for part in out[0, :, 0].split(1 << 21):
        assert bool(((part.float().norm(dim=1) / size - 1).abs() < 2e-3).all())
