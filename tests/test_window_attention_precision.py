"""How exact window_attention_cached is: its probabilities are two terms of 16 bits.

With h half a step of the type, what two roundings leave of a probability is h^2 of
it, or where the second term is below fp16's normal numbers 2^-32 of the row's
largest; the scores' own error (e) is float32's.  Then one rounding of the output.
"""
import pytest
import torch

import test_window_attention as W

DEV = W.DEV

# batch, new tokens, slots, heads, kv heads, values, window, sinks, lengths: one part, and several
CACHES = [(4, 1, 1100, 8, 2, 64, 1000, 4, [1100, 77, 1, 0]), (1, 1, 5000, 4, 2, 64, 4100, 4, [4999]),
          (2, 3, 2500, 4, 2, 128, 2500, 0, [2500, 1700]), (1, 40, 700, 6, 2, 96, 300, 40, [677]), (2, 5, 300, 12, 12, 32, 64, 1, [300, 3])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", W.DTYPES)
@pytest.mark.parametrize("b,t,m,heads,kv,d,window,sinks,lengths", CACHES)
def test_a_cache_is_read_as_exactly_as_the_output_holds(b, t, m, heads, kv, d, window, sinks, lengths, dtype):
    from quant_models import ops

    g = W._gen(m + t)
    q, k, v = W._normal(g, b, t, heads, d, dtype=dtype), W._normal(g, b, m, kv, d, dtype=dtype), W._normal(g, b, m, kv, d, dtype=dtype)
    h, scale = W.HALF[dtype], d ** -0.5
    want, room = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    for x, n in enumerate(lengths):
        if n == 0:
            continue
        i, j = torch.arange(n - t, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        seen = W._seen(i, j, window, sinks, True)
        for y in range(heads):
            vd = v[x, :n, y * kv // heads].double()
            p, e = W._probs(q[x, :, y].double(), k[x, :n, y * kv // heads].double(), seen, scale)
            want[x, :, y] = p @ vd
            room[x, :, y] = (p * (2 * h * h + 2 * e + (n + 8) * W.U) + 2.0 ** -32 * seen) @ vd.abs()
    room += h * (want.abs() + room)
    W._check(ops.window_attention_cached(q, k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), window, sinks), want, room)
