"""linear_int8 with weights that lie as views of other memory do."""
import pytest
import test_int8_linear as base
import torch

DEV = "cuda"
host_path = base.host_path


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40])
@pytest.mark.parametrize("k,left", [(595, 5), (600, 0), (607, 25)])
def test_one_channel_at_the_end_of_its_memory(m, k, left):
    """A single row counts as contiguous whatever its stride: one whose whole 16
    bytes pass its storage's end is copied."""
    from quant_models import ops

    g = base._gen(k)
    memory = torch.randint(-127, 128, (k + left,), device=DEV, generator=g, dtype=torch.int8)
    x = torch.randn(m, k, device=DEV, generator=g)
    scale = torch.rand(1, device=DEV, generator=g)
    for stride in (k + left, 640, 4096):  # the one that a view of wider rows has
        w = memory.as_strided((1, k), (stride, 1), left)
        base._check(ops.linear_int8(x, w, scale), x, w, scale, None)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40])
@pytest.mark.parametrize("n", [1, 5])
def test_rows_far_apart(m, n):
    """Slices of rows more than 2^20 bytes apart are copied too."""
    from quant_models import ops

    g = base._gen(n)
    wide = torch.randint(-127, 128, (n, (1 << 20) + 16), device=DEV, generator=g, dtype=torch.int8)
    x = torch.randn(m, 64, device=DEV, generator=g)
    scale = torch.rand(n, device=DEV, generator=g)
    for w in (wide[:, :64], wide[:, 16:80], wide[:, -64:]):
        base._check(ops.linear_int8(x, w, scale), x, w, scale, None)
