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


# batch, new tokens, slots, heads, kv heads, values, window, sinks, lengths: one part, and several
CACHES = [(2, 1, 300, 4, 2, 64, 200, 2, [300, 77]), (2, 1, 5000, 4, 2, 64, 4100, 4, [4999, 4000]), (2, 3, 2500, 4, 2, 128, 2500, 0, [2500, 1700])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("b,t,m,heads,kv,d,window,sinks,lengths", CACHES)
def test_nan_over_a_cache_is_not_lost_where_parts_are_joined(b, t, m, heads, kv, d, window, sinks, lengths, dtype):
    from quant_models import ops

    g = W._gen(m)
    q, k, v = W._normal(g, b, t, heads, d, dtype=dtype), W._normal(g, b, m, kv, d, dtype=dtype), W._normal(g, b, m, kv, d, dtype=dtype)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want, bound = W._cache_want(q, k, v, lengths, window, sinks, d ** -0.5)
    # a query that is not a number: every score of its row
    one = q.clone()
    one[0, -1, 1, 3] = math.nan
    out = ops.window_attention_cached(one, k, v, lens, window, sinks)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    hit[0, -1, 1] = True
    assert bool(out[hit].isnan().all())
    W._check(torch.where(hit, 0, out), torch.where(hit, 0, want), bound)
    # a stretch of keys that are none, all that some parts see
    lo = max(0, lengths[0] - window)
    one = k.clone()
    one[0, lo:lo + (lengths[0] - lo) * 2 // 3, 0] = math.nan
    out = ops.window_attention_cached(q, one, v, lens, window, sinks)
    hit[:] = False
    hit[0, :, :heads // kv] = True
    assert bool(out[hit].isnan().all())
    W._check(torch.where(hit, 0, out), torch.where(hit, 0, want), bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
def test_nan_is_not_lost_where_sinks_are_divided(dtype):
    from quant_models import ops

    n, heads, kv, d, window, sinks = 1100, 4, 2, 64, 20, 3
    q, k, v, _ = W._inputs(1, n, heads, kv, d, dtype, 11)
    want = W._want(q, k, v, window, sinks, False, d ** -0.5, None)[0]
    one = q.clone()
    one[0, 1, 2, 3] = math.nan
    out = ops.window_attention(one, k, v, window, sinks, causal=False)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    hit[0, 1, 2] = True
    assert bool(out[hit].isnan().all())
    W._check(torch.where(hit, 0, out), torch.where(hit, 0, want[0]), want[1])
    one = k.clone()
    one[0, 300:900, 0] = math.nan  # all that some of the parts see
    out = ops.window_attention(q, one, v, window, sinks, causal=False)
    i = torch.arange(n, device=DEV)
    hit[:] = False
    hit[0, :, :2] = W._seen(i[:, None], i[None, 300:900], window, sinks, False).any(1)[:, None, None]
    assert bool(hit[0, 0, 0].all()) and bool(out[hit].isnan().all())
    W._check(torch.where(hit, 0, out), torch.where(hit, 0, want[0]), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_values_of_no_weight_reach_what_sees_them(causal, dtype):
    """A key 300 above the others: their probabilities are 0 in any type, but a value
    that is not finite among them is seen all the same."""
    from quant_models import ops

    n, heads, kv, d, window, sinks = 200, 4, 2, 64, 30, 2
    q, k, v, _ = W._inputs(1, n, heads, kv, d, dtype, 5)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, 110::50, :, 0] = 300.0  # keys 110 and 160, scores 300
    want = W._want(q, k, v, window, sinks, causal, 0.125, None)[0]
    i = torch.arange(n, device=DEV)
    seen = W._seen(i[:, None], i[None], window, sinks, causal)
    for at, what in ((120, math.inf), (100, math.nan), (1, -math.inf), (158, math.nan)):
        one = v.clone()
        one[0, at, 0, 5] = what
        out = ops.window_attention(q, k, one, window, sinks, causal=causal, scale=0.125)
        hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
        hit[0, :, :2, 5] = seen[:, at][:, None]
        assert not bool(out[hit].isfinite().any())
        W._check(torch.where(hit, 0, out), torch.where(hit, 0, want[0]), want[1])
        for t in (1, 3):  # the last tokens, up to 190
            last, worth = q[:, 190 - t:190].contiguous(), W._cache_want(q[:, 190 - t:190], k, v, [190], window, sinks, 0.125)
            got = ops.window_attention_cached(last, k, one, torch.tensor([190], dtype=torch.int32, device=DEV), window, sinks, scale=0.125)
            near = W._seen(i[190 - t:190], torch.tensor(at, device=DEV), window, sinks, True)
            hit = torch.zeros(got.shape, dtype=torch.bool, device=DEV)
            hit[0, :, :2, 5] = near[:, None]
            assert not bool(got[hit].isfinite().any())
            W._check(torch.where(hit, 0, got), torch.where(hit, 0, worth[0]), worth[1])
