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



class _Conv(nn.Module):
    def __init__(self, device):
        super().__init__()
        g = torch.Generator().manual_seed(3)
        # 1 x 1 kernels have strides of their own kind, a vector none to change
        self.w = nn.Parameter(torch.randn(6, 5, 3, 3, generator=g).to(device))
        self.point = nn.Parameter(torch.randn(8, 6, 1, 1, generator=g).to(device))
        self.b = nn.Parameter(torch.randn(40, generator=g).to(device))


@pytest.mark.gpu
@pytest.mark.parametrize("reload", [False, True])
def test_moments_follow_the_memory_order(reload):
    """Steps before and after model.to(memory_format=...), beside torch's AdamW
    (bounds as in test_optimizer_follows_torch)."""
    import quant_models as qm

    a, b = _Conv(DEV), _Conv(DEV)
    mine, theirs = qm.AdamW(a.parameters(), lr=1e-2), torch.optim.AdamW(b.parameters(), lr=1e-2)
    g = torch.Generator(device=DEV).manual_seed(1)
    k = 0
    for order in (torch.contiguous_format, torch.channels_last, torch.channels_last, torch.contiguous_format):
        a.to(memory_format=order)
        if reload:  # what was saved in one order, loaded into the other
            saved = mine.state_dict()
            mine = qm.AdamW(a.parameters(), lr=5.0)
            mine.load_state_dict(saved)
        for _ in range(2):
            for p, q in zip(a.parameters(), b.parameters()):
                p.grad = torch.randn(p.shape, device=DEV, generator=g)
                q.grad = p.grad.clone()
            mine.step()
            theirs.step()
            k += 1
        for p, q in zip(a.parameters(), b.parameters()):
            assert float((p - q).abs().max()) <= k * 8 * 2.0 ** -24 * (float(q.abs().max()) + 1e-2)
            m, v = mine.state_values(p)
            assert float((m - theirs.state[q]["exp_avg"]).abs().max()) <= k * 4 * 2.0 ** -24 * 5
            assert float((v - theirs.state[q]["exp_avg_sq"]).abs().max()) <= k * 4 * 2.0 ** -24
            assert float(mine.state[p]["step"]) == k


@pytest.mark.gpu
def test_8_bit_states_refuse_another_memory_order():
    import quant_models as qm

    a = _Conv(DEV)
    # the parameter whose order changes is in the second group
    opt = qm.AdamW([{"params": [a.b, a.point]}, {"params": [a.w]}], lr=1e-2, state_bits=8)
    for p in a.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    before = [[t.clone() for t in opt.state_values(p)] for p in a.parameters()]
    old = [p.detach().clone() for p in a.parameters()]
    a.to(memory_format=torch.channels_last)
    for p, t in zip(a.parameters(), before):
        assert all(torch.equal(v, e) for v, e in zip(opt.state_values(p), t))
    with pytest.raises(ValueError, match="memory order"):
        opt.step()
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), old))
    with pytest.raises(ValueError, match="memory order"):
        qm.AdamW([{"params": [a.b, a.point]}, {"params": [a.w]}], state_bits=8).load_state_dict(opt.state_dict())
    a.to(memory_format=torch.contiguous_format)
    opt.step()
    assert all(float(opt.state[p]["step"]) == 2 for p in a.parameters())


@pytest.mark.gpu
def test_a_captured_step_refuses_another_memory_order():
    import quant_models as qm

    a = _Conv(DEV)
    opt = qm.AdamW(a.parameters(), lr=1e-2)
    for p in a.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    a.to(memory_format=torch.channels_last)
    old = [p.detach().clone() for p in a.parameters()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="memory order"):
        with torch.cuda.graph(graph):
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), old))
    opt.step()
    assert all(float(opt.state[p]["step"]) == 2 for p in a.parameters())


def test_8_bit_states_of_another_memory_order_are_not_loaded():
    """On the host: the check comes before anything is taken over."""
    import quant_models as qm

    a = _Conv("cpu")
    opt = qm.AdamW(a.parameters(), state_bits=8)
    step = torch.ones(1)
    for p in a.parameters():
        n = -(-p.numel() // 256)
        opt.state[p] = {"step": step, "exp_avg": torch.ones_like(p, dtype=torch.int8),
                        "exp_avg_sq": torch.ones_like(p, dtype=torch.uint8),
                        "exp_avg_scale": torch.ones(n), "exp_avg_sq_scale": torch.ones(n)}
    saved = opt.state_dict()
    again = qm.AdamW(a.parameters(), lr=0.5, state_bits=8)
    again.load_state_dict(saved)
    assert again.state[a.w]["exp_avg"].dtype == torch.int8
    a.to(memory_format=torch.channels_last)
    fresh = qm.AdamW(a.parameters(), lr=0.5, state_bits=8)
    with pytest.raises(ValueError, match="memory order"):
        fresh.load_state_dict(saved)
    assert fresh.param_groups[0]["lr"] == 0.5 and not fresh.state
