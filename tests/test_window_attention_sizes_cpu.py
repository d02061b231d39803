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


def test_what_no_launch_holds_is_refused():
    """A grid has fewer than 2^32 threads: sizes past it are refused by their numbers,
    before anything is launched."""
    from quant_models import _native as N

    L, at, SHAPE = N.load(), 1 << 20, 2

    def strided(**kw):
        d = _desc(**kw)
        for s in ("q_stride", "k_stride", "v_stride", "out_stride", "grad_stride"):
            getattr(d._obj, s)[:] = (64, 64, 64)
        return d

    def fwd(**kw):
        return L.rpfq_window_attention(strided(M=0, **kw), at, at, at, None, at, None, at, 1 << 60, None)

    def cached(**kw):
        return L.rpfq_window_attention_cached(strided(**kw), at, at, at, at, at, at, 1 << 60, None)

    def stat(**kw):
        return L.rpfq_window_attention_stat_bytes(strided(M=0, **kw))

    # 128 rows of queries a workgroup of 256, 64 of keys
    assert fwd(B=1 << 20, N=1, H=16, KV=16, D=8) == SHAPE and stat(B=1 << 20, N=1, H=16, KV=16, D=8) == 0
    assert stat(B=(1 << 20) - 1, N=1, H=16, KV=16, D=8) > 0 and stat(B=1 << 20, N=1, H=16, KV=4, D=8) > 0
    assert fwd(B=1 << 13, N=1 << 18, H=1, KV=1, D=8) == SHAPE and stat(B=1 << 12, N=1 << 18, H=1, KV=1, D=8) == 0
    assert stat(B=1 << 12, N=(1 << 18) - 64, H=1, KV=1, D=8) > 0
    # over a cache 32 rows of a key head a workgroup of 512, or of 256
    assert cached(B=1, N=1 << 20, H=1024, KV=1, D=64) == SHAPE and cached(B=1, N=1 << 20, H=512, KV=1, D=128) == SHAPE
    assert cached(B=1 << 13, N=1, H=1024, KV=1024, D=64, M=8) == SHAPE
