"""Gradients where hooks on saved tensors (offloading, recomputation) give them back in
another memory order than they were saved in."""
import pytest
import torch

DEV = "cuda"


def _elsewhere(t):
    """The same values, every other element of a larger tensor in another order."""
    order = list(range(t.dim()))[::-1]
    back = torch.empty(*(t.shape[i] for i in order), 2, dtype=t.dtype, device=t.device)[..., 0]
    return back.permute(order).copy_(t)


HOOKS = {"offloaded": lambda: torch.autograd.graph.save_on_cpu(), "elsewhere": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, _elsewhere),
         "packed": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format))}


def _calls():
    """(name, leaves, the call of them), with operands as they lie in larger tensors."""
    from quant_models import ops

    g = torch.Generator(device=DEV).manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    x, res, w = (normal(*s).half().requires_grad_() for s in ((33, 72), (33, 72), (72,)))
    qkv = normal(2, 130, 3, 4, 64).half().requires_grad_()
    lens = torch.tensor([130, 77], dtype=torch.int32, device=DEV)
    wide = torch.randint(0, 500, (2, 130, 6), generator=g, device=DEV)
    freqs = ops.rotary_frequencies((8, 8))
    return [("norm", [x, w], lambda: [ops.rms_norm(x, w)]), ("residual", [x, res, w], lambda: list(ops.rms_norm(x, w, residual=res))),
            ("rotary", [qkv], lambda: list(ops.rotary(qkv.unbind(2)[:2], wide[..., 1:3], freqs, (8, 8)))),
            ("rotary shared", [qkv], lambda: list(ops.rotary(qkv.unbind(2)[:2], wide[1:, :, 4:].expand(2, -1, -1), freqs, (8, 8)))),
            ("rotary one axis", [qkv], lambda: [ops.rotary(qkv[:, :, 1], wide[0, :, 3], freqs)]),
            ("window", [qkv], lambda: [ops.window_attention(*qkv.unbind(2), 20, 2, lengths=lens)]),
            ("window shared", [qkv], lambda: [ops.window_attention(qkv[:, :, 0], qkv[:, :, 1, :1].expand(-1, -1, 2, -1), qkv[:, :, 2, 1::2], 20, causal=False)])]


@pytest.mark.gpu
@pytest.mark.parametrize("hook", sorted(HOOKS))
@pytest.mark.parametrize("name", ["norm", "residual", "rotary", "rotary shared", "rotary one axis", "window", "window shared"])
def test_gradients_through_hooks(name, hook):
    leaves, call = next(c[1:] for c in _calls() if c[0] == name)
    outs = call()
    go = [torch.randn_like(o) for o in outs]
    want = torch.autograd.grad(outs, leaves, go)
    with HOOKS[hook]():
        outs = call()
    got = torch.autograd.grad(outs, leaves, go)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["norm", "residual", "rotary", "window"])
def test_another_tensor_is_refused(name):
    """One of fewer elements, or of another type, is not read as the one that was saved."""
    leaves, call = next(c[1:] for c in _calls() if c[0] == name)
    for change in (lambda t: t[:1], lambda t: t.double() if t.dtype != torch.float64 else t.float()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            outs = call()
        with pytest.raises(RuntimeError, match="another"):
            torch.autograd.grad([o.sum() for o in outs], leaves)


@pytest.fixture(params=["native", "ctypes"])
def host_path(request, monkeypatch):
    if request.param == "ctypes":
        from quant_models import _native

        monkeypatch.setattr(_native, "host", lambda: None)


@pytest.mark.gpu
@pytest.mark.parametrize("hook", sorted(HOOKS))
@pytest.mark.parametrize("bias", [False, True])
def test_the_loss_through_hooks(bias, hook, host_path):
    from quant_models import ops

    g = torch.Generator(device=DEV).manual_seed(1)
    x, w, b = (torch.randn(*s, generator=g, device=DEV).half().requires_grad_() for s in ((40, 64), (90, 64), (90,)))
    target = torch.randint(0, 90, (40,), generator=g, device=DEV)
    leaves = [x, w, b] if bias else [x, w]

    def call():
        return ops.linear_cross_entropy(x, w, target, b if bias else None)

    want = torch.autograd.grad(call(), leaves)
    with HOOKS[hook]():
        loss = call()
    assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(loss, leaves), want))
    for change in (lambda t: t[:1], lambda t: t.double()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            loss = call()
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            torch.autograd.grad(loss, leaves)
