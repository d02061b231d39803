"""Refusals of the int8 layer's, the cross entropy's and AdamW's C entries:
every check is made on the host before any GPU work."""
import ctypes


def lib():
    from quant_models import _native as N

    return N.load(), N


FAKE = 1 << 20  # an aligned non-NULL address; never dereferenced on these paths


def test_quantize_int8_argument_errors():
    L, _ = lib()

    def call(x=FAKE, dt=1, m=4, k=32, codes=FAKE, ld=32, scale=FAKE):
        return L.rpfq_quantize_int8(x, dt, m, k, codes, ld, scale, None)

    assert call(x=None) == 1 and call(codes=None) == 1 and call(scale=None) == 1
    assert call(dt=3) == 5 and call(dt=-1) == 5
    assert call(m=0) == 2 and call(k=0) == 2 and call(ld=31) == 2 and call(m=(1 << 30) + 1) == 2
    assert call(x=FAKE + 1) == 3 and call(scale=FAKE + 2) == 3


def test_linear_int8_argument_errors():
    L, N = lib()

    def call(x=FAKE, dt=1, xs=None, w=FAKE, ld=64, ws=FAKE, b=None, m=300, n=40, k=64, y=FAKE, ydt=1, work=FAKE, nb=1 << 30):
        return L.rpfq_linear_int8(x, dt, xs, w, ld, ws, b, m, n, k, y, ydt, work, nb, None)

    assert call(x=None) == 1 and call(w=None) == 1 and call(ws=None) == 1 and call(y=None) == 1 and call(work=None) == 1
    assert call(xs=FAKE) == 1 and call(dt=N.I8) == 1
    assert call(dt=7) == 5 and call(ydt=3) == 5
    assert call(m=0) == 2 and call(n=0) == 2 and call(k=0) == 2 and call(ld=63) == 2
    assert call(k=131073, ld=131088) == 2 and b"131072" in L.rpfq_last_error()
    assert call(nb=0) == 2
    assert call(x=FAKE + 1) == 3 and call(y=FAKE + 1) == 3 and call(work=FAKE + 16) == 3 and call(b=FAKE + 1) == 3
    size = L.rpfq_linear_int8_workspace_bytes
    assert size(FAKE, 1, 300, 40, 64, FAKE, 64) == 300 * 64 + 1280  # codes and scales, 256-byte pieces
    assert size(FAKE, 1, 8, 40, 64, FAKE, 64) == 0                    # few rows: none
    assert size(FAKE, N.I8, 300, 40, 64, FAKE, 64) == 0
    assert size(FAKE, N.I8, 300, 40, 63, FAKE, 64) > 0                # codes of 63 columns are copied
    assert size(FAKE, 1, 300, 40, 63, FAKE, 63) > size(FAKE, 1, 300, 40, 63, FAKE, 64) > 0
    assert size(FAKE, 1, 0, 40, 64, FAKE, 64) == 0


def _ce(N, M=8, V=100, D=64, dtype=1, bias=1, reduction=1, smoothing=0.0):
    return N.CeDesc(M, V, D, -100, dtype, bias, reduction, smoothing)


def test_linear_cross_entropy_argument_errors():
    L, N = lib()
    size = L.rpfq_linear_cross_entropy_workspace_bytes
    bad = [(dict(M=0), 2), (dict(V=0), 2), (dict(D=0), 2), (dict(M=(1 << 22) + 1), 2), (dict(V=(1 << 22) + 1), 2),
           (dict(D=(1 << 16) + 1), 2), (dict(dtype=3), 5), (dict(bias=4), 5), (dict(reduction=3), 6), (dict(reduction=-1), 6),
           (dict(smoothing=-0.1), 6), (dict(smoothing=1.1), 6), (dict(smoothing=float("nan")), 6)]

    def fwd(d, x=FAKE, w=FAKE, b=None, t=FAKE, loss=FAKE, stat=FAKE, coef=FAKE, work=FAKE, nb=1 << 40):
        return L.rpfq_linear_cross_entropy(ctypes.byref(d) if d else None, x, w, b, t, loss, stat, coef, work, nb, None)

    def bwd(d, x=FAKE, w=FAKE, b=None, t=FAKE, stat=FAKE, coef=FAKE, g=FAKE, gx=FAKE, gw=FAKE, gb=None, work=FAKE, nb=1 << 40):
        return L.rpfq_linear_cross_entropy_grad(ctypes.byref(d) if d else None, x, w, b, t, stat, coef, g, gx, gw, gb, work,
                                                nb, None)

    for kw, code in bad:
        d = _ce(N, **kw)
        assert fwd(d) == code and bwd(d) == code and size(ctypes.byref(d), 0) == 0 == size(ctypes.byref(d), 1), kw
    d = _ce(N)
    assert fwd(None) == 1 and bwd(None) == 1
    for name in ("x", "w", "t", "loss", "stat", "coef", "work"):
        assert fwd(d, **{name: None}) == 1, name
    for name in ("x", "w", "t", "stat", "coef", "g", "work"):
        assert bwd(d, **{name: None}) == 1, name
    assert bwd(d, gx=None, gw=None) == 1
    assert fwd(d, x=FAKE + 8) == 3 and fwd(d, work=FAKE + 128) == 3 and fwd(d, b=FAKE + 1) == 3
    assert bwd(d, gx=FAKE + 1) == 3 and bwd(d, gb=FAKE + 1) == 3
    assert fwd(d, nb=size(ctypes.byref(d), 0) - 1) == 2 and bwd(d, nb=size(ctypes.byref(d), 1) - 1) == 2
    # a piece of dz, not all of it: about 1 GiB whatever V is
    big = _ce(N, M=8192, V=1 << 22, D=64)
    assert (1 << 29) < size(ctypes.byref(big), 1) < (3 << 29)
    # unaligned rows of an odd D are copied, so only the element's alignment counts
    assert fwd(_ce(N, D=65), x=FAKE + 1) == 3


def test_adamw_argument_errors():
    L, N = lib()
    good = N.AdamWHyper(1e-3, 0.9, 0.999, 1e-8, 0.01)

    def table(*rows):
        return (ctypes.c_int64 * (7 * len(rows)))(*[v for r in rows for v in r])

    full = (FAKE, FAKE, FAKE, FAKE, 0, 0, 10)
    small = (FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 10)

    def call(rows=(full,), count=None, dt=0, bits=32, h=good, step=FAKE, work=FAKE):
        return L.rpfq_adamw(table(*rows) if rows else None, len(rows) if count is None else count, dt, bits,
                            ctypes.byref(h) if h else None, step, None, None, None, work, None)

    assert call(h=None) == 1 and call(step=None) == 1 and call(work=None) == 1 and call(rows=(), count=1) == 1
    assert call(count=-1) == 2 and call(dt=3) == 5 and call(bits=16) == 4
    for k in range(4):
        row = list(full)
        row[k] = 0
        assert call(rows=(full, row)) == 1, k
    assert call(rows=(small,)) == 1 and call(rows=(full,), bits=8) == 1 and call(rows=(small[:5] + (0, 10),), bits=8) == 1
    assert call(rows=(full[:6] + (-1,),)) == 2
    assert call(rows=((FAKE + 2,) + full[1:],)) == 3
    for h in ((-1, .9, .9, 0, 0), (1, 1.0, .9, 0, 0), (1, .9, -.1, 0, 0), (1, .9, .9, -1, 0), (1, .9, .9, 0, -1),
              (float("nan"), .9, .9, 0, 0)):
        assert call(h=N.AdamWHyper(*h)) == 6, h
    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int

    def values(c=FAKE, s=FAKE, n=10, o=FAKE, count=1):
        return L.rpfq_adamw_state_values((vp * 1)(c), (vp * 1)(s), (i64 * 1)(n), (i32 * 1)(0), (vp * 1)(o), count, None)

    assert values(c=None) == 1 and values(s=None) == 1 and values(o=None) == 1
    assert values(n=-1) == 2 and values(count=-1) == 2 and values(s=FAKE + 1) == 3
    assert L.rpfq_adamw_state_values(None, None, None, None, None, 1, None) == 1


def test_linear_cross_entropy_takes_at_most_2_39_logits():
    """A launch's threads, two a row and 256 classes, are counted in 32 bits."""
    L, N = lib()
    for backward in (0, 1):
        size = lambda m, v: L.rpfq_linear_cross_entropy_workspace_bytes(ctypes.byref(_ce(N, M=m, V=v)), backward)  # noqa: E731
        assert size(1 << 22, (1 << 17) - 256) > 0 and size(1 << 22, 1 << 17) == 0 == size(1 << 18, 1 << 22)
        assert b"2^39" in L.rpfq_last_error()
