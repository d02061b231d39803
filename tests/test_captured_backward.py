"""A backward pass that is captured while an eager graph of its leaves lives
would end the process where it reaches them: it is refused, however they are
reached, and whatever does not reach them is not."""
import pytest
import torch
import torch.nn as nn

DEV = "cuda"


def _leaves():
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(8, 16, device=DEV, generator=g)
    w = nn.Parameter(torch.randn(40, 16, device=DEV, generator=g))
    return x, w, torch.randint(0, 40, (8,), device=DEV, generator=g)


def _loss(x, w, t, how):
    from quant_models import ops

    if how == "autocast":  # a cast stands between the loss and the leaf
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return ops.linear_cross_entropy(x, w, t)
    return ops.linear_cross_entropy(x, w * 2.0 if how == "scaled" else w, t)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["plain", "autocast", "scaled"])
@pytest.mark.parametrize("inputs", [False, True])
def test_refused_beside_an_eager_graph(how, inputs):
    x, w, t = _leaves()
    alive = _loss(x, w, t, how)
    _loss(x, w, t, how).backward()
    w.grad.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            _loss(x, w, t, how).backward(inputs=[w] if inputs else None)
    assert float(w.grad.abs().max()) == 0
    alive.backward()
    assert float(w.grad.abs().max()) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["plain", "autocast", "scaled"])
def test_captured_where_no_eager_graph_lives(how):
    x, w, t = _leaves()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _loss(x, w, t, how).backward()
    torch.cuda.current_stream().wait_stream(side)
    want = w.grad.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _loss(x, w, t, how).backward()
    for k in range(3):
        w.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w.grad, want)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["plain", "autocast", "scaled"])
def test_gradients_that_are_taken_out(how):
    """grad() of such a leaf is refused as well; of another leaf it is not, and
    then it can be replayed."""
    x, w, t = _leaves()
    alive = _loss(x, w, t, how)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(_loss(x, w, t, how), [w])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        (want,) = torch.autograd.grad(_loss(x.requires_grad_(), w, t, how), [x])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(_loss(x, w, t, how), [x])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    alive.backward()
    assert float(w.grad.abs().max()) > 0
