"""The attention half of a block over many tokens, as a run of its operators: norm
with the residual's addition, qkv layer, rotary positions, attention with a
window, and the same token by token over a cache."""
import pytest
import torch

import test_window_attention as W

DEV = W.DEV


def _parts(seed, b, n, c, heads, dtype):
    g = W._gen(seed)
    x, res = (W._normal(g, b, n, c, dtype=dtype) for _ in range(2))
    norm = (1 + 0.1 * torch.randn(c, generator=g, device=DEV)).float()
    weight = W._normal(g, 3 * c, c, dtype=torch.float32) * c ** -0.5
    positions = torch.stack([torch.arange(n, device=DEV) // 7, torch.arange(n, device=DEV) % 7], -1)
    return x, res, norm, weight, positions


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
def test_eight_bit_block_over_a_padded_batch(dtype):
    """Codes of the norm into the 8-bit qkv layer, its q and k turned where they lie."""
    from quant_models import ops

    b, n, c, heads = 3, 130, 128, 4
    x, res, norm, weight, positions = _parts(1, b, n, c, heads, dtype)
    lengths = [130, 57, 1]
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    codes_w, scale_w = ops.quantize_int8(weight)
    with torch.no_grad():
        codes, scale, h = ops.rms_norm_int8(x, norm, residual=res)
        qkv = ops.linear_int8(codes, codes_w, scale_w, x_scale=scale, out_dtype=dtype).view(b, n, 3, heads, c // heads)
        q, k, v = qkv.unbind(2)
        before = (q.clone(), k.clone())
        ops.rotary((q, k), positions, ops.rotary_frequencies((8, 8)), (8, 8), inplace=True)
        out = ops.window_attention(q, k, v, 40, 1, causal=False, lengths=lens)
    assert torch.equal(h, x + res)
    # 127 steps of a row's and of a weight row's largest value, half a step each, and the type
    y = h.double() * (h.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt() * norm.double()
    want = y @ weight.double().t()
    step = y.abs().amax(-1, keepdim=True) / 254
    room = step * weight.double().abs().sum(1) + (y.abs() + step).sum(-1, keepdim=True) * weight.double().abs().amax(1) / 254
    room = room * (1 + 1e-4) + W.HALF[dtype] * (want.abs() + room) + 1e-5
    plain = torch.stack([*before, v], 2).view(b, n, 3 * c)
    assert bool(((plain.double() - want).abs() <= room).all())
    for now, was in zip((q, k), before):
        assert torch.equal(now, ops.rotary(was, positions, ops.rotary_frequencies((8, 8)), (8, 8)))
    W._check(out, *W._want(q, k, v, 40, 1, False, (c // heads) ** -0.5, lengths)[0])
    assert not bool(out[1, 57:].any()) and not bool(out[2, 1:].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
def test_token_by_token_is_the_whole_sequence(dtype):
    """A prompt at once, then its last tokens one and three at a time over the cache."""
    from quant_models import ops

    b, n, heads, kv, d = 2, 90, 8, 2, 64
    g = W._gen(5)
    q, k, v = (W._normal(g, b, n, e, d, dtype=dtype) for e in (heads, kv, kv))
    positions, freqs = torch.arange(n, device=DEV) + 1000, ops.rotary_frequencies((32,))
    tq, tk = ops.rotary((q, k), positions, freqs)
    whole = ops.window_attention(tq, tk, v, 25, 3)
    _, bound = W._want(tq, tk, v, 25, 3, True, d ** -0.5, None)[0]
    caches = [torch.full((b, 128, kv, d), float("nan"), device=DEV, dtype=dtype) for _ in range(2)]
    for cache, t in zip(caches, (tk, v)):
        cache[:, :70] = t[:, :70]
    at = 70
    while at < n:
        step = 1 if at < 81 else 3
        new = slice(at, at + step)
        nq, nk = ops.rotary((q[:, new], k[:, new]), positions[new], freqs)
        assert torch.equal(nk, tk[:, new])
        caches[0][:, new], caches[1][:, new] = nk, v[:, new]
        at += step
        lens = torch.full((b,), at, dtype=torch.int32, device=DEV)
        out = ops.window_attention_cached(nq, *caches, lens, 25, 3)
        W._check(out, whole[:, new].double(), 2 * bound[:, new])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
def test_gradients_run_through_the_block(dtype):
    """The block's gradients are its operators' own, one behind the other."""
    from quant_models import ops

    b, n, c, heads = 2, 100, 128, 4
    x, res, norm, weight, positions = _parts(9, b, n, c, heads, dtype)
    weight, freqs = weight.to(dtype), ops.rotary_frequencies((8, 8))
    leaves = [t.requires_grad_() for t in (x, res, norm, weight)]
    g = W._gen(10)
    up_out, up_h = W._normal(g, b, n, heads, c // heads, dtype=dtype), W._normal(g, b, n, c, dtype=dtype)

    def layer(y, w):
        return torch.nn.functional.linear(y, w).view(b, n, 3, heads, c // heads)

    y, h = ops.rms_norm(x, norm, residual=res)
    qkv = layer(y, weight)
    q, k, v = qkv.unbind(2)
    tq, tk = ops.rotary((q, k), positions, freqs, (8, 8))
    out = ops.window_attention(tq, tk, v, 30, 1)
    got = torch.autograd.grad([out, h], leaves, [up_out, up_h])

    own = [t.detach().requires_grad_() for t in (tq, tk, v)]
    gq, gk, gv = torch.autograd.grad(ops.window_attention(*own, 30, 1), own, up_out)
    turned = [t.detach().requires_grad_() for t in (q, k)]
    gq, gk = torch.autograd.grad(ops.rotary(tuple(turned), positions, freqs, (8, 8)), turned, [gq, gk])
    flat, w = y.detach().requires_grad_(), weight.detach().requires_grad_()
    gy, gw = torch.autograd.grad(layer(flat, w), [flat, w], torch.stack([gq, gk, gv], 2))
    first = [t.detach().requires_grad_() for t in (x, res, norm)]
    want = torch.autograd.grad(ops.rms_norm(first[0], first[2], residual=first[1]), first, [gy, up_h])
    for a, e in zip(got, (*want, gw)):
        assert torch.equal(a, e)
