"""window_attention, its gradient and its form over a cache, against the definition
in 64 bits.

Bounds, with h half a step of the type and u = 2^-24.  A score is a float32 sum
of D products, so it is off by e = scale (D + 2) u sum|q k| (plus 4 u of its size
for the exponent's argument); a probability is off by e and rounded, h.  The
output divides by the sum of the rounded probabilities: 2 (h + e) sum P|v|, and
its own rounding.  The gradient's probabilities carry the statistic's error (h:
the sum is one of rounded ones) and their own rounding; rowsum(dO O) is off by
what O is.
"""
import ctypes
import math

import pytest
import torch

DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
U = 2.0 ** -24


@pytest.fixture(params=["native", "ctypes"])
def host_path(request, monkeypatch):
    if request.param == "ctypes":
        from quant_models import _native

        monkeypatch.setattr(_native, "host", lambda: None)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _seen(i, j, window, sinks, causal):
    d = i - j
    if causal:
        return (d >= 0) & ((d < window) | (j < sinks))
    return (d.abs() < window) | (j < sinks) | (i < sinks)


def _probs(q, k, seen, scale):
    """(P, bound of a probability's relative error) of one head in 64 bits."""
    s = (q @ k.t()) * scale
    e = scale * (q.shape[1] + 2) * U * (q.abs() @ k.abs().t())
    top = torch.where(seen, s, -math.inf).amax(1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.where(seen, (s - top).exp(), 0.0)
    total = p.sum(1, keepdim=True)
    e = torch.where(seen, e + 4 * U * (s.abs() + top.abs() + 16), 0.0)
    return p / torch.where(total > 0, total, 1.0), e + e.amax(1, keepdim=True)


def _head(q, k, v, seen, scale, h, go=None):
    """Outputs of one head and their bounds, the gradients too where go is given."""
    p, e = _probs(q, k, seen, scale)
    n = k.shape[0]
    out = p @ v
    room = (p * (2 * h + 2 * e + (n + 8) * U)) @ v.abs()
    err = room + h * (out.abs() + room)
    if go is None:
        return [(out, err)]
    pe = p * (2.5 * h + 2 * e + 8 * U)  # of a gradient's probability, rounded
    gv, gv_err = p.t() @ go, pe.t() @ go.abs() + (go.shape[0] + 8) * U * (p.t() @ go.abs())
    dp = go @ v.t()
    dp_err = (q.shape[1] + 2) * U * (go.abs() @ v.abs().t())
    delta, delta_err = (go * out).sum(1, keepdim=True), (go.abs() * (err + (q.shape[1] + 2) * U * out.abs())).sum(1, keepdim=True)
    ds = p * (dp - delta)
    ds_err = pe * (dp - delta).abs() + p * 1.1 * (dp_err + delta_err) + h * ds.abs()
    gq, gq_err = scale * (ds @ k), scale * (ds_err @ k.abs() + (n + 8) * U * (ds.abs() @ k.abs()))
    gk, gk_err = scale * (ds.t() @ q), scale * (ds_err.t() @ q.abs() + (go.shape[0] + 8) * U * (ds.abs().t() @ q.abs()))
    return [(out, err), (gq, gq_err), (gk, gk_err), (gv, gv_err)]


def _want(q, k, v, window, sinks, causal, scale, lengths, go=None):
    """[(values, bounds)] of out, and of the gradients of q, k and v."""
    b, n, heads, d = q.shape
    kv, h = k.shape[2], HALF[q.dtype]
    like = [q, q, k, v] if go is not None else [q]
    res = [(torch.zeros(t.shape, dtype=torch.float64, device=DEV), torch.zeros(t.shape, dtype=torch.float64, device=DEV)) for t in like]
    for x in range(b):
        m = n if lengths is None else min(max(lengths[x], 0), n)
        if m == 0:
            continue
        i = torch.arange(m, device=DEV)
        seen = _seen(i[:, None], i[None], window, sinks, causal)
        for y in range(heads):
            z = y * kv // heads
            one = _head(q[x, :m, y].double(), k[x, :m, z].double(), v[x, :m, z].double(), seen, scale, h,
                        None if go is None else go[x, :m, y].double())
            for at, (w, (val, err)) in enumerate(zip(res, one)):
                head = y if at < 2 else z
                w[0][x, :m, head] += val
                w[1][x, :m, head] += err
    return res


def _check(got, want, bound, rounding=0.0):
    err = (got.double() - want).abs()
    room = bound + rounding * (want.abs() + bound) + TINY[got.dtype]
    assert not bool(got.isnan().any())
    over = float((err / room).max()) if err.numel() else 0.0
    assert over <= 1.0, over


# batch, tokens, heads, kv heads, values, window, sinks, lengths
SHAPES = [(1, 1, 1, 1, 64, 1, 0, None), (2, 5, 4, 1, 8, 2, 1, [5, 0]), (1, 33, 2, 2, 32, 8, 0, None), (2, 64, 6, 2, 128, 1000, 0, [64, 31]),
          (1, 65, 8, 2, 96, 16, 4, None), (3, 127, 3, 1, 40, 31, 70, [127, 1, 96]), (1, 129, 4, 4, 72, 64, 2, None),
          (2, 200, 4, 2, 17, 50, 3, [200, 129]), (1, 300, 16, 4, 128, 65, 16, None), (2, 257, 2, 2, 64, 1, 1, [1000, -3]),
          (1, 450, 2, 1, 104, 130, 200, None), (1, 197, 12, 12, 64, 500, 500, None), (2, 130, 5, 5, 24, 7, 0, [66, 130]),
          # sinks whose far ranges are divided among workgroups
          (1, 1100, 4, 2, 64, 20, 3, None), (2, 900, 4, 1, 32, 9, 65, [900, 333]), (1, 1409, 2, 2, 128, 60, 128, None)]


def _inputs(b, n, heads, kv, d, dtype, seed):
    g = _gen(seed)
    return (_normal(g, b, n, heads, d, dtype=dtype) * 1.5, _normal(g, b, n, kv, d, dtype=dtype), _normal(g, b, n, kv, d, dtype=dtype),
            _normal(g, b, n, heads, d, dtype=dtype) * 0.01)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("b,n,heads,kv,d,window,sinks,lengths", SHAPES)
def test_matches_its_definition(b, n, heads, kv, d, window, sinks, lengths, causal, dtype, host_path):
    from quant_models import ops

    q, k, v, _ = _inputs(b, n, heads, kv, d, dtype, n + d)
    scale = None if n % 2 else 0.3
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32 if n % 2 else torch.int64, device=DEV)
    want = _want(q, k, v, window, sinks, causal, d ** -0.5 if scale is None else scale, lengths)
    if lengths is not None:  # what lies behind the end is not to count
        for t in (q, k, v):
            for x, m in enumerate(lengths):
                t[x, max(m, 0):] = math.nan
    out = ops.window_attention(q, k, v, window, sinks, causal=causal, scale=scale, lengths=lens)
    assert out.dtype == dtype and out.shape == q.shape and out.is_contiguous()
    _check(out, *want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("b,n,heads,kv,d,window,sinks,lengths", SHAPES)
def test_gradients_match_the_formula(b, n, heads, kv, d, window, sinks, lengths, causal, dtype):
    from quant_models import ops

    q, k, v, go = _inputs(b, n, heads, kv, d, dtype, n + d + 1)
    want = _want(q, k, v, window, sinks, causal, d ** -0.5, lengths, go)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    if lengths is not None:
        for t in (q, k, v, go):
            for x, m in enumerate(lengths):
                t[x, max(m, 0):] = math.nan
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.window_attention(*leaves, window, sinks, causal=causal, lengths=lens)
    _check(out.detach(), *want[0])
    grads = torch.autograd.grad(out, leaves, go, retain_graph=True)
    for got, t, w in zip(grads, leaves, want[1:]):
        assert got.dtype == dtype and got.shape == t.shape
        _check(got, *w, rounding=HALF[dtype])
    again = torch.autograd.grad(out, leaves, go, retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))  # sums in a fixed order
    for i in range(3):  # one of them alone
        (only,) = torch.autograd.grad(out, leaves[i], go, retain_graph=True)
        assert torch.equal(only, grads[i])


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_gradients_match_differences(causal):
    """Along a direction, against differences of the definition in 64 bits."""
    from quant_models import ops

    q, k, v, go = _inputs(1, 70, 4, 2, 32, torch.float16, 3)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.window_attention(*leaves, 20, 2, causal=causal), leaves, go)
    bounds = _want(q.detach(), k.detach(), v.detach(), 20, 2, causal, 32 ** -0.5, None, go)[1:]
    g = _gen(9)
    i = torch.arange(70, device=DEV)
    seen = _seen(i[:, None], i[None], 20, 2, causal)

    def loss(at):
        total = 0.0
        for y in range(4):
            p, _ = _probs(at[0][0, :, y], at[1][0, :, y // 2], seen, 32 ** -0.5)
            total += float(((p @ at[2][0, :, y // 2]) * go[0, :, y].double()).sum())
        return total

    for which in range(3):
        base = [t.detach().double() for t in leaves]
        step = torch.randn(base[which].shape, generator=g, device=DEV, dtype=torch.float64)
        eps = 1e-4
        ends = []
        for sign in (eps, -eps):
            moved = list(base)
            moved[which] = base[which] + sign * step
            ends.append(loss(moved))
        slope = (ends[0] - ends[1]) / (2 * eps)
        room = float((step.abs() * (bounds[which][1] + HALF[q.dtype] * 1.01 * bounds[which][0].abs() + TINY[q.dtype])).sum())
        # the differences' own error: third derivatives times eps^2, below 1e-6 of the sizes here
        assert abs(float((grads[which].double() * step).sum()) - slope) <= room + 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("scale_of", [2.0 ** -20, 1.0, 2.0 ** 12])
def test_fp16_gradients_keep_their_range(scale_of):
    """Gradients far from 1: dS and P are carried by powers of two."""
    from quant_models import ops

    q, k, v, go = _inputs(1, 150, 4, 2, 64, torch.float16, 5)
    # a few rows with gradients much larger than the rest
    go = (go * 10).float() * torch.where(torch.arange(150, device=DEV) % 37 == 0, 1.0, 1e-2)[None, :, None, None]
    go = (go * min(scale_of, 2.0 ** 10)).half()
    want = _want(q, k, v, 40, 1, True, 64 ** -0.5, None, go)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.window_attention(*leaves, 40, 1), leaves, go)
    for got, w in zip(grads, want[1:]):
        _check(got, *w, rounding=HALF[torch.float16])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_streams_and_odd_layouts(dtype, host_path):
    from quant_models import ops

    g = _gen(2)
    qkv = _normal(g, 2, 70, 3, 4, 64, dtype=dtype)
    parts = qkv.unbind(2)
    want = ops.window_attention(*(t.contiguous() for t in parts), 20, 2)
    assert torch.equal(ops.window_attention(*parts, 20, 2), want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in parts]
    assert torch.equal(ops.window_attention(*heads_first, 20, 2), want)
    shifted = torch.zeros(qkv.numel() + 1, device=DEV, dtype=dtype)[1:].view_as(qkv).copy_(qkv).unbind(2)
    assert torch.equal(ops.window_attention(*shifted, 20, 2), want)
    values_apart = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in parts]
    assert torch.equal(ops.window_attention(*values_apart, 20, 2), want)
    one = parts[1][:, :, :1]  # a key head that is broadcast, and one that is shared
    same = ops.window_attention(parts[0], one.expand(-1, -1, 4, -1), one.expand(-1, -1, 4, -1), 20, 2)
    assert torch.equal(ops.window_attention(parts[0], one, one, 20, 2), same)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.window_attention(*parts, 20, 2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    for empty in (qkv[:0], qkv[:, :0], qkv[:0, ..., :17]):
        assert ops.window_attention(*empty.unbind(2), 20, 2).shape == empty[:, :, 0].shape
    # a window and sinks past every length, past 32 bits and past 64
    for far in (70, 1 << 33, 1 << 70):
        assert torch.equal(ops.window_attention(*parts, far, far), ops.window_attention(*parts, 70))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_layouts(dtype):
    from quant_models import ops

    g = _gen(6)
    qkv = _normal(g, 2, 70, 3, 4, 64, dtype=dtype).requires_grad_()
    go = _normal(g, 2, 70, 4, 64, dtype=dtype)
    (want,) = torch.autograd.grad(ops.window_attention(*qkv.unbind(2), 20, 2), qkv, go)
    for form in (go.transpose(1, 2).contiguous().transpose(1, 2), go.transpose(2, 3).contiguous().transpose(2, 3),
                 torch.zeros(go.numel() + 3, device=DEV, dtype=dtype)[3:].view_as(go).copy_(go)):
        (got,) = torch.autograd.grad(ops.window_attention(*qkv.unbind(2), 20, 2), qkv, form)
        assert torch.equal(got, want)
    ones = torch.ones_like(go)
    (a,) = torch.autograd.grad(ops.window_attention(*qkv.unbind(2), 20, 2), qkv, ones)
    (b,) = torch.autograd.grad(ops.window_attention(*qkv.unbind(2), 20, 2).sum(), qkv)
    assert torch.equal(a, b)


# batch, new tokens, slots, heads, kv heads, values, window, sinks, lengths
CACHES = [(1, 1, 1, 1, 1, 64, 1, 0, [1]), (3, 1, 40, 4, 1, 128, 16, 4, [40, 1, 23]), (2, 2, 100, 8, 2, 64, 1000, 0, [100, 33]),
          (2, 5, 300, 12, 12, 32, 64, 1, [300, 3]), (1, 40, 200, 6, 2, 96, 30, 40, [177]), (4, 1, 1500, 16, 4, 128, 700, 16, [1500, 900, 12, 0]),
          (2, 3, 777, 4, 4, 40, 100, 0, [5000, -1]), (1, 1, 5000, 2, 1, 17, 4100, 4, [4999]), (9, 1, 513, 4, 2, 72, 33, 33, list(range(1, 514, 64)))]


def _cache_want(q, k, v, lengths, window, sinks, scale):
    b, t, heads, d = q.shape
    out, err = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for x in range(b):
        n = min(max(lengths[x], 0), k.shape[1])
        i, j = torch.arange(n - t, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        if n == 0:
            continue
        seen = _seen(i, j, window, sinks, True)
        for y in range(heads):
            z = y * k.shape[2] // heads
            ((out[x, :, y], err[x, :, y]),) = _head(q[x, :, y].double(), k[x, :n, z].double(), v[x, :n, z].double(), seen, scale, HALF[q.dtype])
    return out, err


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,m,heads,kv,d,window,sinks,lengths", CACHES)
def test_cached_matches_its_definition(b, t, m, heads, kv, d, window, sinks, lengths, dtype, host_path):
    from quant_models import ops

    g = _gen(m + d)
    q, k, v = _normal(g, b, t, heads, d, dtype=dtype) * 1.5, _normal(g, b, m, kv, d, dtype=dtype), _normal(g, b, m, kv, d, dtype=dtype)
    lens = torch.tensor(lengths, dtype=torch.int32 if m % 2 else torch.int64, device=DEV)
    want = _cache_want(q, k, v, lengths, window, sinks, d ** -0.5)
    for x, n in enumerate(lengths):  # slots that no query sees hold anything
        n = min(max(n, 0), m)
        for c in (k, v):
            c[x, n:] = math.nan
            c[x, min(sinks, n):max(min(sinks, n), n - t - window + 1)] = math.nan
    out = ops.window_attention_cached(q, k, v, lens, window, sinks)
    assert out.dtype == dtype and out.shape == q.shape
    _check(out, *want)
    # parts of a cache of other layouts
    both = torch.stack([k, v], 2)
    assert torch.equal(ops.window_attention_cached(q, both[:, :, 0], both[:, :, 1], lens, window, sinks), out)
    first = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v)]
    assert torch.equal(ops.window_attention_cached(q, *first, lens, window, sinks), out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_values_that_are_not_finite_stay_where_they_are_seen(causal, dtype):
    """Infinities and NaN among keys and values reach the queries that see them, and no other."""
    from quant_models import ops

    q, k, v, _ = _inputs(2, 200, 4, 2, 64, dtype, 21)
    want = _want(q, k, v, 30, 2, causal, 0.125, None)
    i = torch.arange(200, device=DEV)
    seen = _seen(i[:, None], i[None], 30, 2, causal)
    for t, at, what in ((v, 77, math.nan), (v, 130, math.inf), (k, 77, math.nan), (v, 199, -math.inf)):
        one = t.clone()
        one[0, at, 0, 5] = what
        out = ops.window_attention(q, one if t is k else k, one if t is v else v, 30, 2, causal=causal)
        hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
        hit[0, :, :2] = seen[:, at][:, None, None]
        if t is v:
            hit[..., :5] = hit[..., 6:] = False
        assert not bool(out[hit].isfinite().any())
        _check(torch.where(hit, 0, out), torch.where(hit, 0, want[0][0]), want[0][1])
    # three new tokens: the last one's values are not the first ones'
    lens = torch.tensor([200, 150], dtype=torch.int32, device=DEV)
    last, worth = q[:, :3].contiguous(), _cache_want(q[:, :3], k, v, [200, 150], 30, 2, 0.125)
    v[0, 199, 0, 5] = math.nan
    out = ops.window_attention_cached(last, k, v, lens, 30, 2)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    hit[0, 2, :2, 5] = True
    assert bool(out[hit].isnan().all())
    _check(torch.where(hit, 0, out), torch.where(hit, 0, worth[0]), worth[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_far_from_zero(dtype):
    """Scores past 2^20, where an exponent's rounding would pass fp16's range."""
    from quant_models import ops

    g = _gen(12)
    q, k, v = (_normal(g, 1, 90, 2, 64, dtype=dtype) for _ in range(3))
    q, k = q * 600, k * 600
    want = _want(q, k, v, 30, 1, True, 4.0, None)
    _check(ops.window_attention(q, k, v, 30, 1, scale=4.0), *want[0])
    lens = torch.tensor([90], dtype=torch.int32, device=DEV)
    _check(ops.window_attention_cached(q[:, -1:].contiguous(), k, v, lens, 30, 1, scale=4.0),
           *_cache_want(q[:, -1:], k, v, [90], 30, 1, 4.0))


@pytest.mark.gpu
def test_captured_step_replays():
    """A training step and a step over a cache in graphs, replayed on other values."""
    from quant_models import ops

    g = _gen(8)
    qkv = _normal(g, 2, 150, 3, 4, 64, dtype=torch.bfloat16).requires_grad_()
    go = _normal(g, 2, 150, 4, 64, dtype=torch.bfloat16)
    lens = torch.tensor([150, 77], dtype=torch.int32, device=DEV)

    def step():
        out = ops.window_attention(*qkv.unbind(2), 40, 2, lengths=lens)
        return [out.detach(), torch.autograd.grad(out, qkv, go)[0]]

    def token():
        return ops.window_attention_cached(qkv[:, :1, 0].detach(), qkv[:, :, 1].detach(), qkv[:, :, 2].detach(), lens, 40, 2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), token()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        got = step()
    with torch.cuda.graph(graphs[1]):
        one = token()
    for turn in range(3):
        with torch.no_grad():
            qkv.copy_(_normal(g, 2, 150, 3, 4, 64, dtype=torch.bfloat16))
            lens.copy_(torch.tensor([150 - turn, 60 + turn], device=DEV))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want, ref = step(), token()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(one, ref)
        del want
    alive = ops.window_attention(*qkv.unbind(2), 40, 2)
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(ops.window_attention(*qkv.unbind(2), 40, 2), qkv, go)
    alive.sum().backward()


@pytest.mark.gpu
def test_once_differentiable():
    from quant_models import ops

    q, k, v, go = _inputs(1, 20, 2, 2, 32, torch.float16, 1)
    q.requires_grad_()
    (grad,) = torch.autograd.grad(ops.window_attention(q, k, v, 5), q, go, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        grad.sum().backward()


@pytest.mark.gpu
def test_refusals(host_path):
    from quant_models import ops

    q, k = torch.randn(2, 5, 4, 32, device=DEV).half(), torch.randn(2, 5, 2, 32, device=DEV).half()
    lens = torch.tensor([5, 5], dtype=torch.int32, device=DEV)
    f, c = ops.window_attention, ops.window_attention_cached
    wide = torch.zeros(1, 2, 1, 136, device=DEV).half()
    bad = [lambda: f(q.cpu(), k, k, 3), lambda: f(q, k.cpu(), k, 3), lambda: f(q, k, k[:, :4], 3), lambda: f(q, k[:, :4], k[:, :4], 3),
           lambda: f(q, k, k.bfloat16(), 3), lambda: f(q, k[..., :16], k[..., :16], 3), lambda: f(q[0], k[0], k[0], 3),
           lambda: f(q[:, :, :3], k, k, 3), lambda: f(k, q, q, 3), lambda: f(wide, wide, wide, 3), lambda: f(q, k, k, 0), lambda: f(q, k, k, -1),
           lambda: f(q, k, k, 3, -1), lambda: f(q, k, k, 2.5), lambda: f(q, k, k, 3, scale=0.0), lambda: f(q, k, k, 3, scale=-1.0),
           lambda: f(q, k, k, 3, scale=math.nan), lambda: f(q, k, k, 3, scale=math.inf), lambda: f(q, k, k, 3, lengths=lens[:1]),
           lambda: f(q, k, k, 3, lengths=lens.float()), lambda: f(q, k, k, 3, lengths=lens.cpu()), lambda: c(q, k, k, None, 3),
           lambda: c(q, k, k, lens[:1], 3), lambda: c(q, k[:1], k[:1], lens, 3), lambda: c(q, k, k[:, :4], lens, 3), lambda: c(q, k, k, lens, 0)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        f(q.float(), k.float(), k.float(), 3)
    with pytest.raises(RuntimeError, match="no gradient"):
        c(q.clone().requires_grad_(), k, k, lens, 3)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.vmap(lambda t: f(t[None], t[None], t[None], 3))(q)


def test_argument_errors():
    from quant_models import _native as N

    L, at = N.load(), 1 << 20

    def desc(cached, **kw):
        d = N.WindowDesc(B=2, N=50, H=4, KV=2, D=64, M=90 if cached else 0, window=9, sinks=1, dtype=1, causal=1, scale=0.125)
        for s in ("q_stride", "k_stride", "v_stride", "out_stride", "grad_stride"):
            getattr(d, s)[:] = (50 * 256, 256, 64)
        for name, v in kw.items():
            if name.endswith("stride"):
                getattr(d, name)[:] = v
            else:
                setattr(d, name, v)
        return ctypes.byref(d)

    def fwd(q=at, k=at, v=at, lens=None, out=at, stat=at, work=at, nb=1 << 40, **kw):
        return L.rpfq_window_attention(desc(False, **kw), q, k, v, lens, out, stat, work, nb, None)

    def grad(q=at, k=at, v=at, lens=None, out=at, go=at, stat=at, gq=at, gk=at, gv=at, work=at, nb=1 << 40, **kw):
        return L.rpfq_window_attention_grad(desc(False, **kw), q, k, v, lens, out, go, stat, gq, gk, gv, work, nb, None)

    def cached(q=at, k=at, v=at, lens=at, out=at, work=at, nb=1 << 40, **kw):
        return L.rpfq_window_attention_cached(desc(True, **kw), q, k, v, lens, out, work, nb, None)

    assert L.rpfq_window_attention(None, at, at, at, None, at, at, at, 1 << 40, None) == 1
    for call in (fwd, grad, cached):
        for name in ("q", "k", "v", "out"):
            assert call(**{name: None}) == 1, (call, name)
            assert call(**{name: at + 8}) == 3, (call, name)
        assert call(dtype=0) == 5 and call(dtype=3) == 5
        for kw in (dict(B=0), dict(N=0), dict(H=0), dict(KV=0), dict(D=0), dict(KV=3), dict(H=1026), dict(D=136), dict(D=63), dict(N=1 << 29),
                   dict(B=1 << 25), dict(B=1 << 23), dict(B=1 << 20, N=1 << 20)):
            assert call(**kw) == 2, (call, kw)
        assert call(window=0) == 6 and call(sinks=-1) == 6 and call(causal=2) == 6
        assert call(scale=0.0) == 6 and call(scale=float("nan")) == 6 and call(scale=float("inf")) == 6
        for name in ("q_stride", "k_stride", "v_stride"):
            assert call(**{name: (1, 256, 64)}) == 3 and call(**{name: (8, 1 << 22, 64)}) == 3 and call(**{name: (8, -8, 64)}) == 3
        assert call(lens=at + 2) == 3
    assert cached(N=1 << 21, H=1024, KV=1) == 2 and fwd(scale=2.0 ** 126) == 6
    assert fwd(M=5) == 2 and grad(M=5) == 2 and cached(M=0) == 2 and cached(M=1 << 29) == 2
    assert fwd(stat=at + 64) == 3 and fwd(out_stride=(8, 4, 8)) == 3
    assert grad(go=None) == 1 and grad(stat=None) == 1 and grad(work=None) == 1 and grad(gq=None, gk=None, gv=None) == 1
    assert grad(go=at + 8) == 3 and grad(gq=at + 8) == 3 and grad(gk=at + 8) == 3 and grad(gv=at + 8) == 3 and grad(work=at + 64) == 3
    assert grad(grad_stride=(8, 4, 8)) == 3
    size = L.rpfq_window_attention_stat_bytes(desc(False))
    assert size == 2 * 4 * 64 * 4 and L.rpfq_window_attention_stat_bytes(desc(False, N=0)) == 0
    need = L.rpfq_window_attention_workspace_bytes
    assert need(desc(False), 0) == 0 and need(desc(False), 1) >= size and need(desc(False, N=0), 1) == 0
    assert grad(nb=need(desc(False), 1) - 1) == 2
    assert cached(lens=None) == 1 and L.rpfq_window_attention_cached_workspace_bytes(desc(True, window=0)) == 0


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A sequence inside a qkv tensor of more than 4 GiB, and caches as long: the last
    rows against the definition on what they see."""
    from quant_models import ops

    n, heads, d, window, sinks = 960_000, 12, 64, 40, 3
    g = _gen(31)
    qkv = torch.randn(1, n, 3, heads, d, generator=g, device=DEV, dtype=torch.float16)
    assert qkv.numel() * 2 > 1 << 32
    q, k, v = qkv.unbind(2)
    tail = 2 * window
    near = torch.cat([torch.arange(sinks, device=DEV), torch.arange(n - tail, n, device=DEV)])
    i = torch.arange(n - window, n, device=DEV)
    seen = _seen(i[:, None], near[None], window, sinks, True)
    want = [_head(q[0, i, y].double(), k[0, near, y].double(), v[0, near, y].double(), seen, d ** -0.5, HALF[q.dtype])[0] for y in range(heads)]
    values, bounds = (torch.stack([w[t] for w in want], 1)[None] for t in range(2))
    with torch.no_grad():
        out = ops.window_attention(q, k, v, window, sinks)
        _check(out[:, -window:], values, bounds)
        assert bool(out[:, :: n // 64].isfinite().all())
        del out
        lens = torch.tensor([n], dtype=torch.int32, device=DEV)
        got = ops.window_attention_cached(q[:, -window:], k, v, lens, window, sinks)
    _check(got, values, bounds)
    # the gradient of the last row: of its own window's keys, and of the sinks
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    go = torch.zeros(1, n, heads, d, device=DEV, dtype=torch.float16)
    go[:, -1] = torch.randn(heads, d, generator=g, device=DEV).half()
    grads = torch.autograd.grad(ops.window_attention(*leaves, window, sinks), leaves, go)
    for y in range(heads):
        one = _head(q[0, -1:, y].double(), k[0, near, y].double(), v[0, near, y].double(), seen[-1:], d ** -0.5, HALF[q.dtype], go[0, -1:, y].double())
        _check(grads[0][0, -1:, y], *one[1], rounding=HALF[q.dtype])
        for got, w in zip(grads[1:], one[2:]):
            _check(got[0, near, y], *w, rounding=HALF[q.dtype])
    assert not bool(grads[1][0, sinks:n - tail:9973].any()) and not bool(grads[0][0, : n - 1 : 9973].any())
