"""window_attention's sizes at the C ABI: workspaces and refusals, which need no GPU."""
import ctypes

import pytest


def _desc(**kw):
    from quant_models import _native as N

    d = N.WindowDesc(B=1, N=1, H=2, KV=1, D=64, M=20000, window=20000, sinks=0, dtype=1, causal=1, scale=0.125)
    for name, v in kw.items():
        setattr(d, name, v)
    return ctypes.byref(d)


@pytest.mark.parametrize("d", [64, 128])
def test_a_window_or_sinks_of_any_size_divide_a_cache_alike(d):
    from quant_models import _native as N

    size = N.load().rpfq_window_attention_cached_workspace_bytes
    want = size(_desc(D=d))
    assert want > 0
    for far in (20000, 1 << 31, 1 << 40, (1 << 63) - 20000, (1 << 63) - 1):
        assert size(_desc(D=d, window=far)) == want
        assert size(_desc(D=d, window=1, sinks=far)) == want
        assert size(_desc(D=d, window=far, sinks=far)) == want


@pytest.mark.parametrize("d", [64, 128])
def test_many_new_tokens_over_a_cache_take_no_workspace(d):
    """Where the rows fill the chip, no float32 sums of them go through memory; the last
    tokens of a few streams over a long cache still go in parts."""
    from quant_models import _native as N

    size = N.load().rpfq_window_attention_cached_workspace_bytes
    for b, n, heads, kv in ((8, 2048, 32, 8), (1, 4096, 16, 4), (1, 1 << 20, 16, 4), (64, 64, 12, 12)):
        assert size(_desc(B=b, N=n, H=heads, KV=kv, D=d)) == 0
    for b, n in ((1, 1), (8, 1), (8, 3), (300, 1), (1, 300)):
        assert size(_desc(B=b, N=n, H=8, KV=2, D=d)) > 0
