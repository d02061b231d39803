"""rotary against its definition in 64 bits, its gradient against the turn back.

The angle is exact to 2^-33 at the positions used here; as a part of a turn it is
rounded to float32 (2^-26 turns, 1.6 2^-24 radians), the cosine and sine are
within 2 2^-24, and each output adds two products: 7 2^-24 (|u| + |v|) in all,
before the one rounding to the type.
"""
import ctypes

import pytest
import torch

DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24


@pytest.fixture(params=["native", "ctypes"])
def host_path(request, monkeypatch):
    if request.param == "ctypes":
        from quant_models import _native

        monkeypatch.setattr(_native, "host", lambda: None)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _freqs(sections):
    from quant_models import ops

    return ops.rotary_frequencies(sections, 10000.0, device=DEV)


def _turned(x, positions, freqs, sections, interleaved, sign=1.0):
    """(values, sizes |u| + |v|) of the definition."""
    p = sum(sections)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(DEV)
    angle = positions.double()[..., axis] * freqs
    angle = (angle if angle.dim() == 3 else angle[None])[:, :, None]
    c, s = angle.cos(), sign * angle.sin()
    xd = x.detach().double()
    want, size = xd.clone(), torch.zeros_like(xd)
    at = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if interleaved else (slice(0, p), slice(p, 2 * p))
    u, v = xd[..., at[0]], xd[..., at[1]]
    want[..., at[0]], want[..., at[1]] = u * c - v * s, v * c + u * s
    size[..., at[0]] = size[..., at[1]] = u.abs() + v.abs()
    return want, size


def _check(got, want, size):
    err = (got.double() - want).abs()
    bound = HALF[got.dtype] * want.abs() + 7 * U * size * (1 + HALF[got.dtype]) + 2.0 ** -25
    assert bool((err <= bound).all()), float((err - bound).max())


# batch, tokens, heads, kv heads, values, sections
SHAPES = [(1, 1, 1, 1, 2, (1,)), (2, 1, 16, 4, 128, (16, 24, 24)), (3, 197, 12, 12, 64, (16, 16)), (2, 33, 3, 1, 64, (6, 10, 10)),
          (1, 300, 4, 2, 40, (20,)), (2, 9, 5, 5, 30, (3, 4, 1, 5)), (1, 17, 2, 2, 96, (24,)), (1, 5, 2, 1, 1024, (512,)),
          (5, 7, 3, 3, 18, (0, 9)), (1, 4000, 1, 1, 32, (8, 8))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,h,kv,d,sections", SHAPES)
def test_matches_its_definition(b, n, h, kv, d, sections, dtype, host_path):
    from quant_models import ops

    g = _gen(n * 7 + d)
    q, k = (torch.randn(b, n, e, d, generator=g, device=DEV).to(dtype) for e in (h, kv))
    freqs = _freqs(sections)
    shared = torch.randint(0, 1 << 20, (n, len(sections)), generator=g, device=DEV)
    own = torch.randint(-5000, 1 << 20, (b, n, len(sections)), generator=g, device=DEV)
    for positions in (shared, own, own.int(), (own % 4096).float() / 8, own.flip(1)[:, :, :].expand(b, n, -1)):
        for inter in (False, True):
            for x in ((q, k), (q,), q):
                out = ops.rotary(x, positions, freqs, sections, interleaved=inter)
                assert type(out) is tuple or x is q
                for a, t in zip(out if type(x) is tuple else (out,), (q, k)):
                    assert a.dtype == dtype and a.shape == t.shape
                    _check(a, *_turned(t, positions, freqs, sections, inter))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_inplace_and_class_tokens(dtype, host_path):
    """Heads inside a qkv tensor, at odd offsets, transposed, in place."""
    from quant_models import ops

    g, sections = _gen(2), (8, 8)
    freqs = _freqs(sections)
    positions = torch.randint(0, 200, (2, 21, 2), generator=g, device=DEV)
    positions[:, 0] = 0
    qkv = torch.randn(2, 21, 3, 4, 32, generator=g, device=DEV).to(dtype)
    want = ops.rotary((qkv[:, :, 0].contiguous(), qkv[:, :, 1].contiguous()), positions, freqs, sections)
    assert torch.equal(want[0][:, 0], qkv[:, 0, 0]) and torch.equal(want[1][:, 0], qkv[:, 0, 1])
    got = ops.rotary((qkv[:, :, 0], qkv[:, :, 1]), positions, freqs, sections)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and all(t.is_contiguous() for t in got)
    shifted = torch.zeros(qkv.numel() + 1, device=DEV, dtype=dtype)[1:].view_as(qkv).copy_(qkv)
    got = ops.rotary((shifted[:, :, 0], shifted[:, :, 1]), positions, freqs, sections)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    heads_first = qkv[:, :, 0].transpose(1, 2).contiguous().transpose(1, 2)  # [B, heads, N, D] in memory
    assert torch.equal(ops.rotary(heads_first, positions, freqs, sections), want[0])
    values_apart = qkv[:, :, 0].transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(ops.rotary(values_apart, positions, freqs, sections), want[0])
    mine = qkv.clone()
    v, before = mine[:, :, 2].clone(), mine._version
    out = ops.rotary((mine[:, :, 0], mine[:, :, 1]), positions, freqs, sections, inplace=True)
    assert out[0].data_ptr() == mine.data_ptr() and mine._version > before
    assert torch.equal(mine[:, :, 0], want[0]) and torch.equal(mine[:, :, 1], want[1]) and torch.equal(mine[:, :, 2], v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rotary(qkv[:, :, 0], positions, freqs, sections)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    assert ops.rotary(qkv[:0, :, 0], positions[:0], freqs, sections).shape == (0, 21, 4, 32)


@pytest.mark.gpu
def test_far_positions_are_exact():
    """A turn of 2^30 steps of 1 radian: as near as one of few steps."""
    from quant_models import ops

    freqs = _freqs((16,))
    x = torch.randn(1, 64, 2, 32, generator=_gen(4), device=DEV)
    far = (1 << 30) + torch.arange(64, device=DEV)[:, None] * 1000003
    want, size = _turned(x, far, freqs, (16,), False)
    err = (ops.rotary(x, far, freqs) - want).abs()
    # the angle itself, formed in 64 bits twice: 2^31 2^-52 radians each
    assert bool((err <= (8 * U + 2 * 2.0 ** -21) * size + 2.0 ** -25).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,h,kv,d,sections", SHAPES[1:6])
@pytest.mark.parametrize("inter", [False, True])
def test_gradients_turn_back(b, n, h, kv, d, sections, inter, dtype):
    from quant_models import ops

    g = _gen(n + d)
    q, k, gq, gk = (torch.randn(b, n, e, d, generator=g, device=DEV).to(dtype) for e in (h, kv, h, kv))
    freqs = _freqs(sections)
    positions = torch.randint(0, 4096, (b, n, len(sections)), generator=g, device=DEV)
    q.requires_grad_(), k.requires_grad_()
    out = ops.rotary((q, k), positions, freqs, sections, interleaved=inter)
    both = torch.autograd.grad(out, [q, k], [gq, gk], retain_graph=True)
    for got, up in zip(both, (gq, gk)):
        _check(got, *_turned(up, positions, freqs, sections, inter, -1.0))
    (only,) = torch.autograd.grad(out[1], k, gk.transpose(1, 3).contiguous().transpose(1, 3), retain_graph=True)
    assert torch.equal(only, both[1])
    one = torch.autograd.grad(out[0], q, torch.ones(1, 1, 1, 1, device=DEV, dtype=dtype).expand_as(q))[0]
    _check(one, *_turned(torch.ones_like(q), positions, freqs, sections, inter, -1.0))
    # against differences: the turn is linear, so a step of 1 is exact up to rounding
    step = torch.randn(q.shape, generator=g, device=DEV, dtype=torch.float64)
    want, size = _turned(step, positions, freqs, sections, inter)
    slope = float((want * gq.double()).sum())
    room = (HALF[dtype] + 8 * U) * float((step.abs() * (both[0].double().abs() + _turned(gq, positions, freqs, sections, inter)[1])).sum())
    assert abs(float((both[0].double() * step).sum()) - slope) <= room + 1e-6


@pytest.mark.gpu
def test_captured_step_replays():
    from quant_models import ops

    g, freqs = _gen(8), _freqs((16, 16))
    q, k = (torch.randn(2, 50, 4, 64, generator=g, device=DEV, requires_grad=True) for _ in range(2))
    positions = torch.randint(0, 900, (50, 2), generator=g, device=DEV)

    def step():
        a, b = ops.rotary((q, k), positions, freqs, (16, 16))
        return torch.autograd.grad(a.square().sum() + (a * b).sum(), [q, k])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        ops.rotary(q.detach(), positions, freqs, (16, 16))
    alive = ops.rotary(q, positions, freqs, (16, 16))
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(ops.rotary(q, positions, freqs, (16, 16)).sum(), q)
    alive.sum().backward()


@pytest.mark.gpu
def test_refusals(host_path):
    from quant_models import ops

    q, k = torch.randn(2, 5, 4, 32, device=DEV), torch.randn(2, 5, 2, 32, device=DEV)
    pos, freqs = torch.zeros(5, 2, dtype=torch.int64, device=DEV), _freqs((8, 8))
    s = (8, 8)
    bad = [lambda: ops.rotary(q.cpu(), pos, freqs, s), lambda: ops.rotary(q, pos.cpu(), freqs, s), lambda: ops.rotary(q, pos, freqs.float(), s),
           lambda: ops.rotary(q, pos, freqs, (8, 4)), lambda: ops.rotary(q, pos, freqs, (8, 8, 0)), lambda: ops.rotary(q, pos[:4], freqs, s),
           lambda: ops.rotary(q, pos.half(), freqs, s), lambda: ops.rotary((q, k[:1]), pos, freqs, s), lambda: ops.rotary((q, k.half()), pos, freqs, s),
           lambda: ops.rotary((q, k, k), pos, freqs, s), lambda: ops.rotary(q[0], pos, freqs, s), lambda: ops.rotary(q, pos, freqs, (-8, 24)),
           lambda: ops.rotary(q[..., :16], pos, freqs, s), lambda: ops.rotary(q, pos, freqs, (4, 4, 4, 2, 2)),
           lambda: ops.rotary((q, k[:, :, :0]), pos, freqs, s), lambda: ops.rotary(q.transpose(2, 3).contiguous().transpose(2, 3), pos, freqs, s, inplace=True),
           lambda: ops.rotary(q[:, :, :1].expand(-1, -1, 4, -1), pos, freqs, s, inplace=True),
           lambda: ops.rotary_frequencies(()), lambda: ops.rotary_frequencies((0, 0)), lambda: ops.rotary_frequencies((4,), -1.0)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        ops.rotary(q.double(), pos, freqs, s)
    with pytest.raises(RuntimeError, match="autograd"):
        ops.rotary(q.clone().requires_grad_(), pos, freqs, s, inplace=True)
    with pytest.raises(RuntimeError, match="positions"):
        ops.rotary(q, pos.float().requires_grad_(), freqs, s)


def test_argument_errors():
    from quant_models import _native as N

    L, at = N.load(), 1 << 20

    def call(q=at, k=at, qo=at, ko=at, pos=at, freqs=at, sections=(8, 8), **kw):
        d = N.RotaryDesc(B=2, N=5, D=32, dtype=1, pos_dtype=0, axes=len(sections))
        d.heads[:] = (4, 2)
        d.sections[:len(sections)] = sections
        for name, v in kw.items():
            if name == "heads":
                d.heads[:] = v
            else:
                setattr(d, name, v)
        return L.rpfq_rotary(ctypes.byref(d), q, k, qo, ko, pos, freqs, None)

    assert L.rpfq_rotary(None, at, at, at, at, at, at, None) == 1
    assert call(q=None) == 1 and call(k=None) == 1 and call(qo=None) == 1 and call(ko=None) == 1 and call(pos=None) == 1 and call(freqs=None) == 1
    assert call(dtype=3) == 5 and call(pos_dtype=3) == 5 and call(pos_dtype=-1) == 5
    assert call(B=0) == 2 and call(N=0) == 2 and call(D=0) == 2 and call(heads=(0, 2)) == 2 and call(heads=(4, -1)) == 2
    assert call(D=1025) == 2 and call(heads=(1025, 0)) == 2 and call(B=1 << 20, N=1 << 11) == 2 and call(sections=(8, 9)) == 2
    assert call(sections=(0, 0)) == 2 and call(sections=(-1, 9)) == 6 and call(axes=0) == 6 and call(axes=5) == 6
    assert call(interleaved=2) == 6 and call(inverse=-1) == 6
    assert call(q=at + 1) == 3 and call(ko=at + 1) == 3 and call(freqs=at + 4) == 3 and call(pos=at + 4) == 3


@pytest.mark.gpu
def test_inplace_refuses_tensors_over_each_other(host_path):
    """q and k that share elements would be turned twice, or not, as it comes."""
    from quant_models import ops

    freqs, pos = _freqs((8,)), torch.arange(6, device=DEV)
    qkv = torch.randn(2, 6, 3, 4, 16, device=DEV)
    packed = torch.randn(2, 6, 8, 16, device=DEV)  # 4 heads of q, 2 of k, 2 of v
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    for pair in ((q, q), (qkv[:, :, 0], qkv[:, :, 0, :2]), (packed[:, :, :4], packed[:, :, 3:5]),
                 (packed[:, :4, :4], packed[:, 2:, :4])):
        with pytest.raises(ValueError, match="inplace"):
            n = pair[0].shape[1]
            ops.rotary(pair, pos[:n], freqs, inplace=True)
    for pair in ((q, k), (packed[:, :, :4], packed[:, :, 4:6]), (qkv[0:1, :, 0], qkv[1:2, :, 0]), (qkv[:, :3, 0], qkv[:, 3:, 0])):
        n = pair[0].shape[1]
        want = ops.rotary(tuple(t.clone() for t in pair), pos[:n], freqs)
        ops.rotary(pair, pos[:n], freqs, inplace=True)
        assert all(torch.equal(t, w) for t, w in zip(pair, want))
