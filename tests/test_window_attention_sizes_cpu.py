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
