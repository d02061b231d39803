"""Dual numbers and functorch's tensors among the arguments that have no gradient of
their own: refused by name, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fa

DEV = "cuda"


@pytest.fixture(params=["native", "ctypes"])
def host_path(request, monkeypatch):
    if request.param == "ctypes":
        from quant_models import _native

        monkeypatch.setattr(_native, "host", lambda: None)


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True])
def test_rotary_refuses_tangents_of_positions_and_frequencies(inplace, host_path):
    from quant_models import ops

    q = torch.randn(1, 5, 2, 8, device=DEV)
    positions, freqs = torch.arange(5.0, device=DEV), ops.rotary_frequencies((4,))
    with fa.dual_level():
        for at, f in ((fa.make_dual(positions, torch.ones_like(positions)), freqs),
                      (positions, fa.make_dual(freqs, torch.ones_like(freqs)))):
            with pytest.raises(RuntimeError, match="rotary has no forward-mode"):
                ops.rotary(q.clone(), at, f, inplace=inplace)
        plain = ops.rotary(q, positions, freqs)  # numbers without a tangent pass within a level
    assert torch.equal(plain, ops.rotary(q, positions, freqs))


@pytest.mark.gpu
def test_functorch_is_refused_by_name(host_path):
    from quant_models import ops

    q = torch.randn(1, 5, 2, 8, device=DEV)
    h = torch.randn(1, 5, 2, 32, device=DEV).half()
    freqs = ops.rotary_frequencies((4,))
    lens = torch.tensor([[5], [3]], dtype=torch.int32, device=DEV)
    for call, arg in ((lambda p: ops.rotary(q, p, freqs), torch.randn(3, 5, device=DEV)),
                      (lambda f: ops.rotary(q, torch.arange(5, device=DEV), f), torch.randn(3, 4, device=DEV).double()),
                      (lambda n: ops.window_attention(h, h, h, 3, lengths=n), lens),
                      (lambda n: ops.window_attention_cached(h, h, h, n, 3), lens)):
        with pytest.raises(RuntimeError, match="functorch"):
            torch.func.vmap(call)(arg)
