"""window_attention, its gradient and its form over a cache where scores lie far
from zero: up to 2^26, exact in float32 by their making (a large product that all
share and whole steps beside it), so that no bound grows with their size.

What is left of a probability's error: the exponent (S - top) scale2 - lg, with
|S - top| scale2 <= 44, a shift or lg of 28 at most, four roundings and scale2's
own, log 2 x 2^-24 x 3 x 72 together; the exponential and the logarithm of a sum,
an ulp each, 2^-23 and 28 x 2^-23.  E = 256 x 2^-24 is above their sum.
"""
import math

import pytest
import torch

import test_window_attention as W

DEV = W.DEV
E = 256 * W.U


@pytest.fixture
def exact_scores(monkeypatch):
    def probs(q, k, seen, scale):
        s = (q @ k.t()) * scale
        top = torch.where(seen, s, -math.inf).amax(1, keepdim=True)
        top = torch.where(top > -math.inf, top, 0.0)
        p = torch.where(seen, (s - top).exp(), 0.0)
        total = p.sum(1, keepdim=True)
        return p / torch.where(total > 0, total, 1.0), torch.where(seen, E, 0.0)

    monkeypatch.setattr(W, "_probs", probs)


def _far(b, n, m, heads, kv, d, dtype, size, kind, seed):
    """(q, k, v, grad, scale): scores size + unit c, and with scale = 1 / unit
    whole c beside a constant; unit: the spacing of float32 at `size`."""
    g = W._gen(seed)
    unit = max(1.0, abs(size) * 2.0 ** -23)
    root = 2.0 ** (math.frexp(abs(size))[1] // 2)
    q, k = torch.zeros(b, n, heads, d, device=DEV), torch.zeros(b, m, kv, d, device=DEV)
    q[..., 0], k[..., 0] = size / root, root
    q[..., d // 2 + 1] = unit
    if kind == "near":
        k[..., d // 2 + 1] = torch.randint(0, 6, k.shape[:3], generator=g, device=DEV).float()
    elif kind == "dominant":
        k[..., d // 2 + 1] = torch.where(torch.randint(0, 40, k.shape[:3], generator=g, device=DEV) == 0, 24.0, 0.0)
    v, go = W._normal(g, b, m, kv, d, dtype=dtype), W._normal(g, b, n, heads, d, dtype=dtype) * 0.01
    assert torch.equal(q.to(dtype).float(), q) and torch.equal(k.to(dtype).float(), k)
    return q.to(dtype), k.to(dtype), v, go, 1.0 / unit


def _sharp(want, bound, dtype):
    """Zeros in the place of the answer would fail, and not at a few values."""
    assert float((want.abs() > bound + W.TINY[dtype]).double().mean()) > 0.25


# batch, tokens, heads, kv heads, values, window, sinks, causal, lengths
SHAPES = [(1, 300, 4, 2, 64, 70, 2, True, None), (2, 150, 4, 1, 128, 40, 1, False, [150, 77]),
          # sinks whose far ranges are divided among workgroups
          (1, 1100, 4, 2, 64, 20, 3, False, None), (1, 900, 4, 1, 32, 9, 40, True, None)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("kind", ["tied", "near", "dominant"])
@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 19, 2.0 ** 22, -2.0 ** 22, 2.0 ** 26])
@pytest.mark.parametrize("b,n,heads,kv,d,window,sinks,causal,lengths", SHAPES)
def test_gradients_of_far_scores(b, n, heads, kv, d, window, sinks, causal, lengths, size, kind, dtype, exact_scores):
    from quant_models import ops

    q, k, v, go, scale = _far(b, n, n, heads, kv, d, dtype, size, kind, n)
    want = W._want(q, k, v, window, sinks, causal, scale, lengths, go)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.window_attention(*leaves, window, sinks, causal=causal, scale=scale, lengths=lens)
    full = slice(0, 1)  # a sequence without padding
    _sharp(want[0][0][full], want[0][1][full], dtype)
    if kind != "dominant":  # there most keys have next to no gradient
        _sharp(want[3][0][full], want[3][1][full], dtype)
    W._check(out.detach(), *want[0])
    for got, w in zip(torch.autograd.grad(out, leaves, go), want[1:]):
        W._check(got, *w, rounding=W.HALF[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_equal_keys_weigh_alike_whatever_their_scores(causal, dtype):
    """Every key the same: each probability is one over their number, though the scores
    (sums of rounded products up to 2^24) are rounded themselves."""
    from quant_models import ops

    n, heads, kv, d, window = 200, 4, 2, 64, 50
    g = W._gen(4)
    q, k, v = (W._normal(g, 1, n, h, d, dtype=dtype) * s for h, s in ((heads, 600), (kv, 600), (kv, 1)))
    k = k[:, :1].expand(-1, n, -1, -1).contiguous()
    go = W._normal(g, 1, n, heads, d, dtype=dtype)
    h = W.HALF[dtype]
    i = torch.arange(n, device=DEV)
    seen = W._seen(i[:, None], i[None], window, 0, causal).double()
    p = seen / seen.sum(1, keepdim=True)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.window_attention(*leaves, window, causal=causal, scale=4.0)
    gv = torch.autograd.grad(out, leaves[2], go)[0]
    for y in range(kv):
        vd = v[0, :, y].detach().double()
        for x in range(heads // kv * y, heads // kv * (y + 1)):
            room = (2 * h + 2 * E + n * W.U) * (p @ vd.abs())
            W._check(out[0, :, x].detach(), p @ vd, room + h * ((p @ vd).abs() + room))
        god = go[0, :, heads // kv * y:heads // kv * (y + 1)].double()
        each, size = (torch.einsum("ij,ihd->jd", p, t) for t in (god, god.abs()))
        W._check(gv[0, :, y], each, (2.5 * h + 2 * E + 2 * n * W.U) * size, rounding=h)


# batch, new tokens, slots, heads, kv heads, values, window, sinks, lengths
CACHES = [(2, 1, 300, 4, 2, 64, 200, 2, [300, 77]), (1, 1, 5000, 4, 1, 64, 4000, 4, [4990]), (2, 3, 2500, 4, 2, 128, 2500, 0, [2500, 1700])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("kind", ["tied", "near", "dominant"])
@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 22, -2.0 ** 22, 2.0 ** 26])
@pytest.mark.parametrize("b,t,m,heads,kv,d,window,sinks,lengths", CACHES)
def test_far_scores_over_a_cache(b, t, m, heads, kv, d, window, sinks, lengths, size, kind, dtype, exact_scores):
    from quant_models import ops

    q, k, v, _, scale = _far(b, t, m, heads, kv, d, dtype, size, kind, m)
    want = W._cache_want(q, k, v, lengths, window, sinks, scale)
    _sharp(*want, dtype)
    W._check(ops.window_attention_cached(q, k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), window, sinks, scale=scale), *want)


def test_what_goes_with_the_statistic():
    """stat, desc.top and desc.rests go together, and are checked before anything is launched."""
    import ctypes

    from quant_models import _native as N

    L, at = N.load(), 1 << 20

    def desc(top, rests):
        d = N.WindowDesc(B=2, N=50, H=4, KV=2, D=64, window=9, sinks=1, dtype=1, causal=1, scale=0.125, top=top, rests=rests)
        for s in ("q_stride", "k_stride", "v_stride", "out_stride", "grad_stride"):
            getattr(d, s)[:] = (50 * 256, 256, 64)
        return ctypes.byref(d)

    def fwd(top, rests, stat):
        return L.rpfq_window_attention(desc(top, rests), at, at, at, None, at, stat, at, 1 << 40, None)

    def grad(top, rests):
        return L.rpfq_window_attention_grad(desc(top, rests), at, at, at, None, at, at, at, at, at, at, at, 1 << 40, None)

    assert fwd(None, at, at) == 1 and fwd(at, None, at) == 1 and fwd(at, at, None) == 1 and fwd(at, None, None) == 1 and fwd(None, at, None) == 1
    assert fwd(at + 64, at, at) == 3 and fwd(at, at + 8, at) == 3
    assert grad(None, at) == 1 and grad(at, None) == 1 and grad(at + 64, at) == 3 and grad(at, at + 8) == 3
