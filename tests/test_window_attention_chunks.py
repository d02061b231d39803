"""A piece of a prompt over a cache: many new tokens at once."""
import pytest
import torch

import test_window_attention as W

DEV = W.DEV

# batch, new tokens, slots, heads, kv heads, values, window, sinks, lengths
CHUNKS = [(2, 300, 2000, 8, 2, 64, 1500, 4, [2000, 1333]), (8, 260, 1500, 8, 4, 128, 900, 0, [1500, 260, 261, 777, 100, 1499, 0, 900]),
          (1, 700, 1700, 12, 4, 96, 40, 2, [1650])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("b,t,m,heads,kv,d,window,sinks,lengths", CHUNKS)
def test_chunks_match_the_definition(b, t, m, heads, kv, d, window, sinks, lengths, dtype):
    from quant_models import ops

    g = W._gen(t + d)
    q, k, v = W._normal(g, b, t, heads, d, dtype=dtype) * 1.5, W._normal(g, b, m, kv, d, dtype=dtype), W._normal(g, b, m, kv, d, dtype=dtype)
    want = W._cache_want(q, k, v, lengths, window, sinks, d ** -0.5)
    for x, n in enumerate(lengths):
        for c in (k, v):
            c[x, n:] = float("nan")
    out = ops.window_attention_cached(q, k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), window, sinks)
    W._check(out, *want)


@pytest.mark.gpu
def test_more_rows_to_join_than_workgroups():
    """A million rows in parts: each is joined, the last among them."""
    from quant_models import ops

    b, m, heads, d = 33000, 1300, 32, 8
    g = W._gen(1)
    q = W._normal(g, b, 1, heads, d, dtype=torch.float16)
    k, v = (W._normal(g, 1, m, 1, d, dtype=torch.float16).expand(b, -1, -1, -1) for _ in range(2))
    lens = torch.full((b,), m, dtype=torch.int32, device=DEV)
    out = ops.window_attention_cached(q, k, v, lens, m)
    at = torch.tensor([0, 1, 32767, 32768, b - 1], device=DEV)
    W._check(out[at], *W._cache_want(q[at], k[:5], v[:5], [m] * 5, m, 0, d ** -0.5))
    assert bool(out.isfinite().all()) and bool(out.any(-1).all())
