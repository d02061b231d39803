"""adamw and adamw_state_values against the formulas in 64 bits.

float32 states: each of the two sums rounds three times, the parameter's
update about ten times: bounds of 4 and 12 half steps of the magnitudes that
are added.  8-bit states: the codes are those of the definition, exactly.
"""
import math

import pytest
import torch

DEV = "cuda"


@pytest.fixture(autouse=True, params=["native", "ctypes"])
def host_path(request, monkeypatch):
    """Every test on the native host path and on the Python one behind it."""
    if request.param == "ctypes":
        from quant_models import _native

        monkeypatch.setattr(_native, "host", lambda: None)


HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E24 = 2.0 ** -24
SIZES = [(1,), (3,), (255,), (256,), (257,), (64, 33), (4096,), (4097,), (1000, 13), (5, 0), (3, 5, 7), (70000,)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tensors(dtype, bits, seed, sizes=SIZES, count=1):
    g = _gen(seed)
    made = {k: [] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales")}
    for size in sizes * count:
        p = torch.randn(size, device=DEV, generator=g)
        made["params"].append((p * 0.05).to(dtype))
        made["grads"].append((torch.randn(size, device=DEV, generator=g) * 10.0 ** torch.randint(-4, 1, size, device=DEV, generator=g)).to(dtype))
        if bits == 32:
            made["exp_avgs"].append(torch.randn(size, device=DEV, generator=g) * 1e-2)
            made["exp_avg_sqs"].append(torch.rand(size, device=DEV, generator=g) * 1e-3)
        else:
            n = p.numel()
            made["exp_avgs"].append(torch.randint(-127, 128, size, device=DEV, generator=g, dtype=torch.int8))
            made["exp_avg_sqs"].append(torch.randint(0, 256, size, device=DEV, generator=g, dtype=torch.uint8))
            made["exp_avg_scales"].append(torch.rand(-(-n // 256), device=DEV, generator=g) * 1e-2)
            made["exp_avg_sq_scales"].append(torch.rand(-(-n // 256), device=DEV, generator=g) * 1e-3)
    if bits == 32:
        del made["exp_avg_scales"], made["exp_avg_sq_scales"]
    return made


def _values(codes, scales):
    s = scales.double().repeat_interleave(256)[:codes.numel()].view(codes.shape)
    c = codes.double()
    return c.abs() * c / 127 ** 2 * s if codes.dtype == torch.int8 else c ** 4 / 255 ** 4 * s


def _encode(m, v):
    """Codes and scales of 64-bit states, from the definition."""
    def blocks(t):
        flat = torch.zeros(-(-t.numel() // 256) * 256, dtype=torch.float64, device=DEV)
        flat[:t.numel()] = t.reshape(-1)
        return flat.view(-1, 256)

    out = []
    for t, top, power, dtype in ((m, 127, 2, torch.int8), (v, 255, 4, torch.uint8)):
        b = blocks(t)
        s = torch.zeros(0, device=DEV)
        if b.numel():  # the power of two at or above the largest
            part, e = torch.frexp(b.abs().amax(1))
            s = torch.where(part > 0, torch.ldexp(torch.ones_like(part), e - (part == 0.5).int()).clamp_min(2.0 ** -126), 0.0).float()
        ratio = b.abs() / torch.where(s > 0, s, 1.0).double()[:, None]
        edges = ((torch.arange(top, device=DEV, dtype=torch.float64) + 0.5) / top) ** power
        c = torch.bucketize(ratio, edges).double()
        if power == 4:
            c = torch.where((b > 0) & (c == 0) & (s > 0)[:, None], 1.0, c)
        out += [(c * b.sign()).reshape(-1)[:t.numel()].view(t.shape).to(dtype), s]
    return out


def _step(old, t, lr, betas, eps, wd, scale=1.0):
    """(m, v, p, bound of p) of every tensor in 64 bits."""
    b1, b2 = betas
    for i, (p, g) in enumerate(zip(old["params"], old["grads"])):
        p, g = p.double(), g.double() / scale
        if "exp_avg_scales" in old:
            m, v = _values(old["exp_avgs"][i], old["exp_avg_scales"][i]), _values(old["exp_avg_sqs"][i], old["exp_avg_sq_scales"][i])
        else:
            m, v = old["exp_avgs"][i].double(), old["exp_avg_sqs"][i].double()
        m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        up = lr / (1 - b1 ** t) * m1 / ((v1 / (1 - b2 ** t)).sqrt() + eps)
        size = lr / (1 - b1 ** t) * (b1 * m.abs() + (1 - b1) * g.abs()) / ((v1 / (1 - b2 ** t)).sqrt() + eps)
        want = p * (1 - lr * wd) - up
        half = HALF[old["params"][i].dtype]
        tiny = 2.0 ** -25 if old["params"][i].dtype == torch.float16 else 2.0 ** -140
        bound = half * want.abs() + 12 * E24 * (1 + half) * (p.abs() + size) + tiny
        yield m, g, v, m1, v1, want, bound


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 11])  # 11: more tensors than one launch takes
def test_step_matches_its_definition(dtype, bits, count):
    from quant_models import ops

    new = _tensors(dtype, bits, 3 + count, count=count)
    step = torch.full((1,), 6.0, device=DEV)
    for k in range(3):
        old = {n: [x.clone() for x in v] for n, v in new.items()}
        ops.adamw(step=step, lr=2e-3, betas=(0.9, 0.99), eps=1e-7, weight_decay=0.1, **new)
        assert float(step) == 7.0 + k
        for i, (m, g, v, m1, v1, want, bound) in enumerate(_step(old, 7 + k, 2e-3, (0.9, 0.99), 1e-7, 0.1)):
            err = (new["params"][i].double() - want).abs()
            assert bool((err <= bound).all()), (i, float((err - bound).max()))
            assert torch.equal(new["grads"][i], old["grads"][i])
            if bits == 32:
                assert bool(((new["exp_avgs"][i].double() - m1).abs() <= 4 * E24 * (m.abs() + g.abs())).all())
                assert bool(((new["exp_avg_sqs"][i].double() - v1).abs() <= 5 * E24 * (v + g * g)).all())
            else:
                cm, sm, cv, sv = _encode(m1, v1)
                assert torch.equal(new["exp_avg_scales"][i], sm) and torch.equal(new["exp_avg_sq_scales"][i], sv)
                assert torch.equal(new["exp_avgs"][i], cm) and torch.equal(new["exp_avg_sqs"][i], cv)
    if bits == 8:
        got = ops.adamw_state_values(new["exp_avgs"] + new["exp_avg_sqs"], new["exp_avg_scales"] + new["exp_avg_sq_scales"])
        codes, scales = new["exp_avgs"] + new["exp_avg_sqs"], new["exp_avg_scales"] + new["exp_avg_sq_scales"]
        for a, c, s in zip(got, codes, scales):
            want = _values(c, s)
            assert a.shape == c.shape and bool(((a.double() - want).abs() <= 1.01 * E24 * want.abs() + 2.0 ** -149).all())


@pytest.mark.gpu
@pytest.mark.parametrize("b1,b2", [(0.9, 0.999), (0.5, 0.5), (0.0, 0.99), (0.95, 0.9)])
def test_codes_over_many_magnitudes(b1, b2):
    """400,000 elements: blocks of zeros, without a gradient, of gradients that
    nearly cancel the moment, of tiny and huge scales, single large values."""
    from quant_models import ops

    g = _gen(21)
    blocks, n = 1600, 1600 * 256 - 37
    c = torch.randint(-127, 128, (n,), device=DEV, generator=g, dtype=torch.int8)
    u = torch.randint(0, 256, (n,), device=DEV, generator=g, dtype=torch.uint8)
    s = torch.exp2(torch.randint(-60, 8, (blocks,), device=DEV, generator=g).float())
    r = torch.exp2(torch.randint(-100, 12, (blocks,), device=DEV, generator=g).float())
    of = torch.arange(n, device=DEV) // 256
    kind = of % 8
    grad = torch.randn(n, device=DEV, generator=g) * s[of] * 10.0 ** torch.randint(-3, 3, (n,), device=DEV, generator=g)
    c[kind == 0], u[kind == 0], grad[kind == 0] = 0, 0, 0
    grad[kind == 1] = 0
    m = _values(c, s)
    near = (-m * (b1 / (1 - b1)) * (1 + 1e-4 * torch.randn(n, device=DEV, generator=g))).float()
    grad[kind == 2] = near[kind == 2]
    c[kind == 3], u[kind == 3] = 0, 0
    c[(kind == 4) & (torch.arange(n, device=DEV) % 256 != 9)] = 0
    grad[kind == 5] = grad[kind == 5] * 1e-25
    s[5::16], r[5::16], u[kind == 6] = 2.0 ** -126, 2.0 ** -126, 1
    p = torch.zeros(n, device=DEV)
    cm, sm, cv, sv = _encode(b1 * _values(c, s) + (1 - b1) * grad.double(),
                             b2 * _values(u, r) + (1 - b2) * grad.double() * grad.double())
    ops.adamw([p], [grad], [c], [u], torch.ones(1, device=DEV), betas=(b1, b2), exp_avg_scales=[s], exp_avg_sq_scales=[r])
    assert torch.equal(s, sm) and torch.equal(r, sv)
    assert torch.equal(c, cm) and torch.equal(u, cv)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_first_steps_from_zero_states(bits):
    """New states are zeros; 20 steps of a noisy gradient stay near 64-bit AdamW
    (8 bits: the moments are off by at most half a code a step)."""
    from quant_models import ops

    g = _gen(9)
    n = 3000
    p = torch.randn(n, device=DEV, generator=g)
    state = {"exp_avgs": [torch.zeros(n, device=DEV, dtype=torch.float32 if bits == 32 else torch.int8)],
             "exp_avg_sqs": [torch.zeros(n, device=DEV, dtype=torch.float32 if bits == 32 else torch.uint8)]}
    if bits == 8:
        state |= {"exp_avg_scales": [torch.zeros(12, device=DEV)], "exp_avg_sq_scales": [torch.zeros(12, device=DEV)]}
    step, q, m, v = torch.zeros(1, device=DEV), p.double(), 0.0, 0.0
    for k in range(1, 21):
        grad = torch.randn(n, device=DEV, generator=g) * 0.01 + 0.01
        ops.adamw([p], [grad], step=step, lr=1e-2, **state)
        m, v = 0.9 * m + 0.1 * grad.double(), 0.999 * v + 0.001 * grad.double() ** 2
        q = q * (1 - 1e-4) - 1e-2 / (1 - 0.9 ** k) * m / ((v / (1 - 0.999 ** k)).sqrt() + 1e-8)
    assert float(step) == 20
    # a step moves by about lr; 8 bits: codes of m are 2 / 127 of its block's
    # largest apart at most, so each of 20 updates is off by a few hundredths of lr
    assert float((p.double() - q).abs().max()) <= (1e-5 if bits == 32 else 20 * 1e-2 * 0.1)


@pytest.mark.gpu
def test_small_second_moments_keep_a_code():
    """An element far below its block's largest: v's code is 1, not 0, and a
    block of zeros stays zeros."""
    from quant_models import ops

    n = 512
    grad = torch.zeros(n, device=DEV)
    grad[0], grad[1] = 1.0, 1e-9
    c, s = [torch.zeros(n, device=DEV, dtype=torch.int8)], [torch.zeros(2, device=DEV)]
    u, r = [torch.zeros(n, device=DEV, dtype=torch.uint8)], [torch.zeros(2, device=DEV)]
    p = torch.zeros(n, device=DEV)
    ops.adamw([p], [grad], c, u, torch.zeros(1, device=DEV), lr=1.0, weight_decay=0.0, exp_avg_scales=s, exp_avg_sq_scales=r)
    # m = 0.1 under s = 2^-3: 127 sqrt(0.8) = 113.6; v = 0.001 under 2^-9: 255 0.512^(1/4) = 215.7
    assert c[0][:3].tolist() == [114, 0, 0] and u[0][:3].tolist() == [216, 1, 0]
    assert s[0].tolist() == [2.0 ** -3, 0.0] and r[0].tolist() == [2.0 ** -9, 0.0]
    assert bool((c[0][256:] == 0).all()) and bool((u[0][256:] == 0).all()) and float(s[0][1]) == 0 == float(r[0][1])
    assert bool(torch.isfinite(p).all()) and bool((p[2:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_gradient_scaler_and_device_learning_rate(bits):
    from quant_models import ops

    a, b = _tensors(torch.float32, bits, 4), _tensors(torch.float32, bits, 4)
    before = {k: [t.clone() for t in v] for k, v in a.items()}
    step = torch.full((1,), 3.0, device=DEV)
    ops.adamw(step=step, found_inf=torch.ones(1, device=DEV), **a)
    assert float(step) == 3 and all(torch.equal(x, y) for k in a for x, y in zip(a[k], before[k]))
    scaled = dict(a, grads=[g * 1024 for g in a["grads"]])
    ops.adamw(step=step, lr=torch.tensor(0.5, device=DEV), grad_scale=torch.full((), 1024.0, device=DEV),
              found_inf=torch.zeros(1, device=DEV), **scaled)
    ops.adamw(step=(other := torch.full((1,), 3.0, device=DEV)), lr=0.5, **b)
    assert float(step) == 4 == float(other)
    for k in a:
        if k != "grads":
            assert all(torch.equal(x, y) for x, y in zip(a[k], b[k]))


@pytest.mark.gpu
def test_gradients_that_are_not_finite():
    """NaN stays with its element; 8-bit states: with its block's states."""
    from quant_models import ops

    for bits in (32, 8):
        t = _tensors(torch.float32, bits, 8, [(1000,)])
        t["grads"][0][300] = float("nan")
        ops.adamw(step=torch.ones(1, device=DEV), **t)
        assert int(torch.isnan(t["params"][0]).sum()) == 1 and bool(torch.isnan(t["params"][0][300]))
        if bits == 8:
            assert torch.isnan(t["exp_avg_scales"][0]).tolist() == [False, True, False, False]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_tensors_and_guards(bits):
    """Views at odd offsets of one buffer: the same bits, and nothing between
    the tensors is written."""
    from quant_models import ops

    t = _tensors(torch.float32, bits, 5)
    moved, flats = {}, {}
    for k, tensors in t.items():
        gap = 3
        flat = torch.full((sum(x.numel() + gap for x in tensors) + gap,), 77, device=DEV, dtype=tensors[0].dtype)
        at, views = gap, []
        for x in tensors:
            views.append(flat[at:at + x.numel()].view(x.shape))
            views[-1].copy_(x)
            at += x.numel() + gap
        moved[k], flats[k] = views, flat
    ops.adamw(step=torch.ones(1, device=DEV), **t)
    ops.adamw(step=torch.ones(1, device=DEV), **moved)
    for k in t:
        assert all(torch.equal(a, b) for a, b in zip(t[k], moved[k])), k
        inside = torch.zeros_like(flats[k], dtype=torch.bool)
        for v in moved[k]:
            o = v.storage_offset()
            inside[o:o + v.numel()] = True
        assert bool((flats[k][~inside] == 77).all()), k


@pytest.mark.gpu
def test_captured_steps_count_on():
    from quant_models import ops

    for bits in (32, 8):
        a, b = _tensors(torch.float32, bits, 6), _tensors(torch.float32, bits, 6)
        s1, s2, lr = torch.zeros(1, device=DEV), torch.zeros(1, device=DEV), torch.full((1,), 1e-2, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.adamw(step=s1, lr=lr, **a)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.adamw(step=s1, lr=lr, **a)
        ops.adamw(step=s2, lr=1e-2, **b)
        for k in range(4):
            lr.fill_(1e-2 / (k + 1))
            for x, y in zip(a["grads"], b["grads"]):
                x.mul_(0.9)
                y.mul_(0.9)
            graph.replay()
            ops.adamw(step=s2, lr=float(lr), **b)
            torch.cuda.synchronize()
            assert float(s1) == float(s2) == k + 2
            for n in a:
                assert all(torch.equal(x, y) for x, y in zip(a[n], b[n])), n


@pytest.mark.gpu
def test_changed_weights_are_told_by_their_version():
    from quant_models import ops

    t = _tensors(torch.float32, 32, 7, [(64,), (65,)])
    was = [p._version for p in t["params"]]
    ops.adamw(step=torch.zeros(1, device=DEV), **t)
    assert all(p._version > v for p, v in zip(t["params"], was))


@pytest.mark.gpu
def test_refusals():
    from quant_models import ops

    step = torch.zeros(1, device=DEV)
    good = lambda: _tensors(torch.float32, 32, 1, [(8,), (9,)])  # noqa: E731
    small = _tensors(torch.float32, 8, 1, [(8,), (9,)])

    def change(k, i, f, base=None):
        t = {n: list(v) for n, v in (base or good()).items()}
        t[k][i] = f(t[k][i])
        return t

    bad = [dict(good(), grads=good()["grads"][:1]), change("grads", 0, lambda x: x[:4]), change("exp_avgs", 1, lambda x: x[:4]),
           change("params", 0, lambda x: torch.randn(8, 2, device=DEV)[:, 0]), change("grads", 1, lambda x: x.cpu()),
           {k: v for k, v in small.items() if k != "exp_avg_scales"}, change("exp_avg_scales", 0, lambda x: x[:0], small),
           {k: [] for k in good()}]
    twice = good()
    twice["params"][1], twice["grads"][1] = twice["params"][0], twice["grads"][0]
    twice["exp_avgs"][1], twice["exp_avg_sqs"][1] = torch.zeros(8, device=DEV), torch.zeros(8, device=DEV)
    for t in bad + [twice]:
        with pytest.raises(ValueError):
            ops.adamw(step=step, **t)
    for t in (change("grads", 0, lambda x: x.half()), change("exp_avgs", 0, lambda x: x.half()),
              change("params", 0, lambda x: x.double()), change("exp_avgs", 0, lambda x: x.float(), small)):
        with pytest.raises(TypeError):
            ops.adamw(step=step, **t)
    for kw in ({"step": step.double()}, {"step": step.cpu()}, {"step": torch.zeros(2, device=DEV)},
               {"step": step, "found_inf": torch.zeros(2, device=DEV)}, {"step": step, "lr": torch.zeros(1)}):
        with pytest.raises(ValueError):
            ops.adamw(**kw, **good())
    for kw in ({"lr": -1.0}, {"betas": (1.0, 0.9)}, {"eps": -1.0}, {"weight_decay": -0.1}, {"lr": math.nan}):
        with pytest.raises(RuntimeError):
            ops.adamw(step=step, **kw, **good())
    assert float(step) == 0
    with pytest.raises(ValueError):
        ops.adamw_state_values([step], [step])
    assert ops.adamw_state_values([], []) == []


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_overlapping_tensors_are_refused(bits):
    from quant_models import ops

    made = _tensors(torch.float32, bits, 1, [(8,), (9,)])
    wide = torch.zeros(16, device=DEV)
    step = torch.zeros(1, device=DEV)
    for k in ("params", "exp_avgs"):
        t = {n: list(v) for n, v in made.items()}
        wide_k = wide.to(t[k][0].dtype)
        t[k] = [wide_k[:8], wide_k[7:]]
        with pytest.raises(ValueError, match="overlap"):
            ops.adamw(step=step, **t)
        t[k] = [wide_k[:8], wide_k[8:][:9].new_zeros(9)]
        ops.adamw(step=step, **t)


@pytest.mark.gpu
def test_states_made_in_inference_mode():
    from quant_models import ops

    a, b = (_tensors(torch.float32, 32, 2, [(8,), (300,)]) for _ in range(2))
    with torch.inference_mode():
        a["exp_avgs"] = [t.clone() for t in a["exp_avgs"]]
    for t in (a, b):
        ops.adamw(step=torch.zeros(1, device=DEV), **t)
    assert all(torch.equal(p, q) for p, q in zip(a["params"] + a["exp_avgs"], b["params"] + b["exp_avgs"]))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_2_31_elements(bits):
    """The end and the middle of a tensor are the bits of a step on those alone."""
    from quant_models import ops

    n, part = (1 << 31) + (1 << 20), 4096 * 25
    g = _gen(3)
    t = {"params": [torch.randn(n, device=DEV, generator=g, dtype=torch.bfloat16)],
         "grads": [torch.randn(n, device=DEV, generator=g, dtype=torch.bfloat16)]}
    kinds = (torch.float32, torch.float32) if bits == 32 else (torch.int8, torch.uint8)
    t["exp_avgs"], t["exp_avg_sqs"] = ([torch.zeros(n, device=DEV, dtype=k)] for k in kinds)
    if bits == 8:
        t["exp_avg_scales"], t["exp_avg_sq_scales"] = ([torch.zeros(n // 256, device=DEV)] for _ in range(2))
    at = (0, 1 << 30, (1 << 31) - 4096, n - part)
    cut = lambda v, a: v[a // (n // v.numel()):(a + part) // (n // v.numel())]  # noqa: E731
    alone = [{k: [cut(v[0], a).clone()] for k, v in t.items()} for a in at]
    for call in [t] + alone:
        for _ in range(2):
            ops.adamw(step=torch.zeros(1, device=DEV), lr=0.1, **call)
    for a, call in zip(at, alone):
        for k, v in call.items():
            assert torch.equal(cut(t[k][0], a), v[0]), k
