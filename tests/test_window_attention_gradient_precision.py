"""How exact window_attention's gradients are.

rowsum(dO O) is float32's: O goes into it with what its rounding left, and P went
into O as two 16-bit terms.  Up to 8,192 rows P and dS are two terms in the
gradients' products too: every rounding but the results' own is h^2 of a value, h
half a step of the type, so the bounds of test_window_attention hold with h^2 in
the place of h, and one rounding behind them.

Over more rows dS (P) is one term: each product's error is as large as a result's own
rounding, relative to it, and of random sign, so their sum over the keys has the
variance that the result's rounding has: together sqrt(2) of it, over thousands
of rows 1.5 at most.
"""
import pytest
import torch

import test_window_attention as W

DEV = W.DEV


def _gradients(b, n, heads, kv, d, window, sinks, lengths, causal, dtype, seed):
    from quant_models import ops

    q, k, v, go = W._inputs(b, n, heads, kv, d, dtype, seed)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.window_attention(*leaves, window, sinks, causal=causal, lengths=lens)
    return [out.detach(), *torch.autograd.grad(out, leaves, go)], (q.detach(), k.detach(), v.detach()), go


# batch, tokens, heads, kv heads, values, window, sinks, lengths
FEW = [(2, 5, 4, 1, 8, 2, 1, [5, 2]), (1, 3, 16, 4, 96, 31, 1, None), (8, 2, 12, 12, 64, 40, 0, None), (1, 33, 2, 2, 32, 8, 0, None),
       (2, 64, 6, 2, 128, 1000, 0, [64, 31]), (3, 127, 3, 1, 40, 31, 70, [127, 1, 96]), (2, 257, 4, 2, 64, 60, 1, None),
       # sinks whose far ranges are divided among workgroups
       (1, 1100, 4, 2, 64, 20, 3, None)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("b,n,heads,kv,d,window,sinks,lengths", FEW)
def test_few_rows_are_as_exact_as_the_type(b, n, heads, kv, d, window, sinks, lengths, causal, dtype, monkeypatch):
    h = W.HALF[dtype]
    got, qkv, go = _gradients(b, n, heads, kv, d, window, sinks, lengths, causal, dtype, n + d)
    monkeypatch.setitem(W.HALF, dtype, h * h)
    for x, w in zip(got, W._want(*qkv, window, sinks, causal, d ** -0.5, lengths, go)):
        W._check(x, *w, rounding=h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("b,n,heads,kv,d,window,sinks", [(8, 300, 12, 12, 64, 6, 0), (6, 260, 16, 4, 128, 40, 2), (16, 197, 8, 2, 32, 300, 1)])
def test_many_rows_lose_no_more_than_another_rounding(b, n, heads, kv, d, window, sinks, causal, dtype):
    got, qkv, go = _gradients(b, n, heads, kv, d, window, sinks, None, causal, dtype, n)
    for x, (want, _) in zip(got, W._want(*qkv, window, sinks, causal, d ** -0.5, None, go)):
        least = float((want.to(dtype).double() - want).norm())
        assert float((x.double() - want).norm()) <= 1.5 * least
