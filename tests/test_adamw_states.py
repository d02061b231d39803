"""AdamW's states where they come from elsewhere or lie otherwise: runs that
torch.optim.AdamW began, and parameters whose memory order changes."""
import pytest
import torch
import torch.nn as nn

DEV = "cuda"


def _torch_run(dtype, device, steps=2):
    """Parameters after some steps of torch's AdamW, their optimizer, a generator."""
    g = torch.Generator(device=device).manual_seed(7)
    params = [nn.Parameter(torch.randn(s, device=device, generator=g).to(dtype)) for s in ((33, 17), (300,), (8, 3, 5, 5))]
    opt = torch.optim.AdamW(params, lr=1e-2)
    for _ in range(steps):
        for p in params:
            p.grad = torch.randn(p.shape, device=device, generator=g).to(dtype)
        opt.step()
    return params, opt, g


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_moments_of_a_torch_run_become_float32(dtype):
    """torch keeps the moments of fp16 and bf16 parameters in their type."""
    import quant_models as qm

    params, theirs, _ = _torch_run(dtype, "cpu")
    mine = qm.AdamW(params, lr=5.0)
    mine.load_state_dict(theirs.state_dict())
    for p in params:
        for name in ("exp_avg", "exp_avg_sq"):
            assert mine.state[p][name].dtype == torch.float32 and theirs.state[p][name].dtype == dtype
            assert torch.equal(mine.state[p][name], theirs.state[p][name].float())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_torch_run_goes_on(dtype):
    """The step after loading, from the definition in 64 bits on the loaded
    moments: half a step of the parameter's type, and of float32 eight times."""
    import quant_models as qm

    params, theirs, g = _torch_run(dtype, DEV)
    mine = qm.AdamW(params, lr=5.0, state_bits=8)
    mine.load_state_dict(theirs.state_dict())
    want = []
    for p in params:
        s = theirs.state[p]
        p.grad = torch.randn(p.shape, device=DEV, generator=g).to(dtype)
        gd = p.grad.double()
        m, v = 0.9 * s["exp_avg"].double() + 0.1 * gd, 0.999 * s["exp_avg_sq"].double() + 0.001 * gd * gd
        step = 1e-2 * (m / (1 - 0.9 ** 3)) / ((v / (1 - 0.999 ** 3)).sqrt() + 1e-8)
        want.append((p.detach().double() * (1 - 1e-2 * 1e-2) - step, step, m, v))
    mine.step()
    for p, (q, step, m, v) in zip(params, want):
        bound = torch.finfo(dtype).eps / 2 * q.abs() * 1.01 + 8 * 2.0 ** -24 * (q.abs() + step.abs()) + 2.0 ** -25
        # torch's fp16 run leaves an element where 0.001 g^2 rounded to 0 in its first
        # step (|g| below 0.005): m / (0 + 1e-8), whose 1e-8 is 0 in fp16 too
        fine = torch.isfinite(q)
        assert torch.equal(fine, torch.isfinite(p)) and float(fine.double().mean()) > 0.98
        assert bool(((p.detach().double() - q).abs() <= bound)[fine].all())
        s = mine.state[p]
        assert float(s["step"]) == 3
        # m and v: two rounded products, one rounded sum and 1 - b rounded; the
        # terms of m may cancel
        for got, e, terms in ((s["exp_avg"], m, 0.2 * float(p.grad.abs().max())), (s["exp_avg_sq"], v, 0.0)):
            assert got.dtype == torch.float32
            assert bool(((got.double() - e).abs() <= 4 * 2.0 ** -24 * (e.abs() + terms)).all())
