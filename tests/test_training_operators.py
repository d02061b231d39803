"""The new operators where the framework uses them: the AdamW optimizer, a
classifier's loss without its logits, the 8-bit baseline of a model, and the
three of them in one run.  What is compared is computed by torch on the same
values; each bound says what the two sides round differently."""
import copy
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

DEV = "cuda"


def _model(name="rpfq_vit_tiny_patch16_224_q", device=DEV, **kw):
    import quant_models as qm

    torch.manual_seed(3)
    m = qm.create_model(name, num_classes=10, img_size=32, quant_method_u="complex_phase_v2",
                        quant_method_w="complex_phase_v2", enable_act_quant=True, **kw).to(device)
    for p in m.parameters():  # a head of zeros would hide its inputs
        if p.dim() == 2 and float(p.detach().abs().max()) == 0:
            nn.init.normal_(p, std=0.02)
    return m


# ---------------------------------------------------------------------------
# host only
# ---------------------------------------------------------------------------
def test_int8_linear_on_the_host():
    import quant_models as qm

    torch.manual_seed(0)
    layer = nn.Linear(37, 11)
    q = qm.Int8Linear.from_linear(layer)
    x = torch.randn(2, 5, 37)
    with torch.no_grad():
        y, want = q(x), layer(x)
    # half a code of x and of w, and their product
    bound = (x.abs().amax(-1, keepdim=True) / 254 * layer.weight.abs().sum(1)
             + x.abs().sum(-1, keepdim=True) * layer.weight.abs().amax(1) / 254) * 1.01
    assert y.shape == (2, 5, 11) and bool(((y - want).abs() <= bound + 1e-6).all())
    assert q.codes.shape == (11, 48) and bool((q.codes[:, 37:] == 0).all())
    half = copy.deepcopy(q).half()  # a cast leaves codes, scales and bias
    assert half.weight_scale.dtype == torch.float32 and torch.equal(half.weight_scale, q.weight_scale)
    other = qm.Int8Linear(37, 11)
    other.load_state_dict(q.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), y)
    with pytest.raises(RuntimeError, match="no gradient"):
        q(x.clone().requires_grad_())
    with pytest.raises(ValueError):
        q(torch.randn(2, 36))
    with pytest.raises(ValueError):
        qm.Int8Linear(0, 4)
    nan = x.clone()
    nan[0, 1, 3] = math.nan
    with torch.no_grad():
        y2 = q(nan)
    assert bool(torch.isnan(y2[0, 1]).all()) and int(torch.isnan(y2).sum()) == 11


def test_to_int8_replaces_and_skips():
    import quant_models as qm
    from quant_models.inference import to_int8

    m = _model(device="cpu")
    n = sum(isinstance(x, nn.Linear) for x in m.modules())
    assert to_int8(m, skip=("head", "blocks.1")) == n - 5
    assert isinstance(m.head, nn.Linear) and isinstance(m.blocks[1].mlp.fc1, nn.Linear)
    assert isinstance(m.blocks[0].mlp.fc1, qm.Int8Linear)
    assert to_int8(m) == 5


def test_optimizer_and_loss_refusals_on_the_host():
    import quant_models as qm

    p = nn.Parameter(torch.zeros(4))
    for kw in ({"lr": -1.0}, {"eps": -1.0}, {"weight_decay": -1.0}, {"betas": (0.9, 1.0)}, {"state_bits": 16}):
        with pytest.raises(ValueError):
            qm.AdamW([p], **kw)
    opt = qm.AdamW([p])
    opt.step()  # no gradients: nothing to do
    p.grad = torch.zeros(4)
    with pytest.raises(ValueError, match="device"):
        opt.step()
    with pytest.raises(TypeError):
        qm.classifier_loss(nn.Linear(4, 4), torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64))


# ---------------------------------------------------------------------------
# optimizer
# ---------------------------------------------------------------------------
def _pair(bits, seed=0):
    """Two copies of parameters in two groups, one of them channels last, one fp16."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = [torch.randn(s, device=DEV, generator=g) for s in ((33, 17), (300,), (8, 3, 5, 5), (1,), (700,))]
    make[2] = make[2].contiguous(memory_format=torch.channels_last)
    a = [nn.Parameter(t.clone(memory_format=torch.preserve_format)) for t in make]
    b = [nn.Parameter(t.clone()) for t in make]
    return a, b, g


@pytest.mark.gpu
def test_optimizer_follows_torch():
    """30 steps beside torch's float32 AdamW: both round each step's update to
    float32 a few times (30 x 8 half steps of the parameter and of lr)."""
    import quant_models as qm

    a, b, g = _pair(32)
    groups = lambda p: [{"params": p[:2], "lr": 3e-3}, {"params": p[2:], "weight_decay": 0.0}]  # noqa: E731
    mine, theirs = qm.AdamW(groups(a), lr=1e-3, weight_decay=0.1), torch.optim.AdamW(groups(b), lr=1e-3, weight_decay=0.1)
    for k in range(30):
        for i, (p, q) in enumerate(zip(a, b)):
            grad = torch.randn(p.shape, device=DEV, generator=g)
            # one parameter is left out of some steps, as torch leaves it out
            p.grad, q.grad = (None, None) if i == 1 and k % 3 == 0 else (grad.clone(), grad.clone())
        mine.step()
        theirs.step()
    for p, q in zip(a, b):
        assert p.stride() == p.detach().clone(memory_format=torch.preserve_format).stride()
        assert float((p - q).abs().max()) <= 30 * 8 * 2.0 ** -24 * (float(q.abs().max()) + 3e-3)
        s, t = mine.state[p], theirs.state[q]
        assert float(s["step"]) == float(t["step"])
        assert float((s["exp_avg"] - t["exp_avg"]).abs().max()) <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_survives_saving(bits):
    """state_dict through torch.save: the next steps are the same bits."""
    import io

    import quant_models as qm

    a, _, g = _pair(bits)
    opt = qm.AdamW(a, state_bits=bits)
    grads = [[torch.randn(p.shape, device=DEV, generator=g) for p in a] for _ in range(4)]

    def go(params, opt, gs):
        for grad in gs:
            for p, x in zip(params, grad):
                p.grad = x.clone()
            opt.step()

    go(a, opt, grads[:2])
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    b = [nn.Parameter(p.detach().clone(memory_format=torch.preserve_format)) for p in a]
    again = qm.AdamW(b, state_bits=bits)
    again.load_state_dict(torch.load(file, weights_only=True))
    go(a, opt, grads[2:])
    go(b, again, grads[2:])
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for name, v in opt.state[p].items():
            w = again.state[q][name]
            assert v.dtype == w.dtype and torch.equal(v, w), name
        for v, w in zip(opt.state_values(p), again.state_values(q)):
            assert v.shape == p.shape and v.dtype == torch.float32 and torch.equal(v, w)
    # one count, so one launch, for all of them after loading too
    assert len({id(again.state[q]["step"]) for q in b}) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_under_the_gradient_scaler(bits):
    """A step with an infinite gradient is left out, scale and all."""
    import quant_models as qm

    torch.manual_seed(1)
    net = nn.Linear(40, 30).to(DEV)
    opt = qm.AdamW(net.parameters(), state_bits=bits)
    scaler = torch.amp.GradScaler("cuda", init_scale=256.0, growth_interval=1000)
    x = torch.randn(16, 40, device=DEV)
    for k in range(3):
        opt.zero_grad(set_to_none=True)
        scaler.scale(net(x).square().mean()).backward()
        before = [p.detach().clone() for p in net.parameters()]
        if k == 1:
            net.weight.grad[3, 3] = math.inf
        scaler.step(opt)
        scaler.update()
        moved = [not torch.equal(p, q) for p, q in zip(net.parameters(), before)]
        assert moved == ([False, False] if k == 1 else [True, True])
    assert float(opt.state[net.weight]["step"]) == 2 and scaler.get_scale() == 128.0


@pytest.mark.gpu
def test_optimizer_refusals_and_closure():
    import quant_models as qm

    p = nn.Parameter(torch.randn(8, 6, device=DEV)[:, ::2])
    p.grad = torch.ones(8, 3, device=DEV)
    with pytest.raises(ValueError, match="gaps"):
        qm.AdamW([p]).step()
    q = nn.Parameter(torch.randn(5, device=DEV))
    opt = qm.AdamW([q], lr=torch.full((1,), 0.1, device=DEV))

    def closure():
        opt.zero_grad()
        loss = q.square().sum()
        loss.backward()
        return loss

    before = q.detach().clone()
    loss = opt.step(closure)
    assert float(loss.detach()) == pytest.approx(float(before.square().sum())) and not torch.equal(q, before)
    # a first step moves every element by about lr
    assert float(((q - before).abs() - 0.1).abs().max()) <= 0.1 * 0.01 * float(before.abs().max()) + 1e-5


@pytest.mark.gpu
def test_optimizer_makes_packed_layers_pack_again():
    """Evaluation after a step runs on the new weights."""
    import quant_models as qm

    m = _model()
    x = torch.randn(4, 3, 32, 32, device=DEV)
    m.eval()
    with torch.no_grad():
        before = m(x)
    opt = qm.AdamW(m.parameters(), lr=1e-2)
    m.train()
    m(x).sum().backward()
    opt.step()
    m.eval()
    with torch.no_grad():
        after = m(x)
        fresh = _model()
        fresh.load_state_dict(m.state_dict())
        assert not torch.equal(after, before) and torch.equal(after, fresh.eval()(x))


# ---------------------------------------------------------------------------
# loss
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rpfq_vit_tiny_patch16_224_q", "rpfq_deit_tiny_patch16_224_q",
                                  "rpfq_swin_tiny_patch4_window7_224_q"])
@pytest.mark.parametrize("amp", [False, True])
def test_classifier_loss_is_the_models_loss(name, amp):
    """Loss and gradients beside F.cross_entropy(model(x)): float32 on both
    sides (sums in another order, 1e-5), or fp16 logits that torch rounds
    (2^-11 of each) and this does not."""
    import quant_models as qm

    m = _model(name).train()
    x = torch.randn(6, 3, 32, 32, device=DEV)
    t = torch.tensor([1, 9, -100, 0, 3, 3], device=DEV)

    def run(f):
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.float16, enabled=amp):
            loss = f()
        loss.backward()
        return loss.detach(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}

    a, ga = run(lambda: qm.classifier_loss(m, x, t, label_smoothing=0.1))
    b, gb = run(lambda: F.cross_entropy(m(x), t, label_smoothing=0.1))
    tol = 2.0 ** -9 if amp else 1e-5
    assert abs(float(a) - float(b)) <= tol * (1 + abs(float(b)))
    assert ga.keys() == gb.keys()
    heads = [n for n in ga if n.startswith("head")]
    assert heads
    for n in heads:  # the head's own gradients: nothing is quantized behind them
        assert float((ga[n] - gb[n]).norm()) <= (2.0 ** -8 if amp else 1e-4) * float(gb[n].norm()) + 1e-7, n
    if not amp:
        for n in ga:
            assert float((ga[n] - gb[n]).norm()) <= 1e-3 * float(gb[n].norm()) + 1e-6, n


# ---------------------------------------------------------------------------
# 8-bit models, and all of it in one run
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_int8_model_on_the_device(dtype):
    """Every layer of a model in 8 bits: each Int8Linear gives what its
    definition gives for the input it sees."""
    import quant_models as qm
    from quant_models.inference import prepare_inference, to_int8

    m = _model().eval()
    n = sum(isinstance(x, nn.Linear) for x in m.modules())
    assert to_int8(m) == n
    prepare_inference(m, DEV, dtype)
    seen = []
    for layer in m.modules():
        if isinstance(layer, qm.Int8Linear):
            assert layer.weight_scale.dtype == torch.float32 and layer.codes.is_cuda
            layer.register_forward_hook(lambda mod, args, out: seen.append((mod, args[0], out)))
    with torch.no_grad():
        y = m(torch.randn(3, 3, 32, 32, device=DEV, dtype=dtype))
    assert y.shape == (3, 10) and y.dtype == dtype and len(seen) == n and bool(torch.isfinite(y).all())
    half = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    for mod, x, out in seen:
        xd = x.double().cpu()
        top = xd.abs().amax(-1, keepdim=True)
        q = torch.round(127 * xd / torch.where(top > 0, top, 1.0))
        prod = (q @ mod.weight_codes.double().cpu().t()) * (top / 127).float().double() * mod.weight_scale.double().cpu()
        want = prod if mod.bias is None else prod + mod.bias.double().cpu()
        size = prod.abs() + (0 if mod.bias is None else mod.bias.double().cpu().abs())
        assert bool(((out.double().cpu() - want).abs() <= half * want.abs() + 5 * 2.0 ** -24 * size + 2.0 ** -25).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_train_step_and_answer(bits):
    """A head trained on the loss without logits, stepped with AdamW and then
    answered in 8 bits, beside the same in torch's operations: the weights
    after three steps within the update's size where a gradient's sign is not
    in doubt, the answers within what 8 bits allow."""
    import quant_models as qm
    from quant_models import ops

    g = torch.Generator(device=DEV).manual_seed(2)
    head, ref = nn.Linear(96, 500).to(DEV), nn.Linear(96, 500).to(DEV)
    ref.load_state_dict(head.state_dict())
    opt, opt_ref = qm.AdamW(head.parameters(), lr=1e-3, state_bits=bits), torch.optim.AdamW(ref.parameters(), lr=1e-3)
    for _ in range(3):
        x = torch.randn(200, 96, device=DEV, generator=g)
        t = torch.randint(0, 500, (200,), device=DEV, generator=g)
        for layer, o, f in ((head, opt, lambda: ops.linear_cross_entropy(x, head.weight, t, head.bias)),
                            (ref, opt_ref, lambda: F.cross_entropy(ref(x), t))):
            o.zero_grad(set_to_none=True)
            f().backward()
            o.step()
    assert torch.equal(opt.state[head.weight]["step"], torch.full((1,), 3.0, device=DEV))
    diff = (head.weight - ref.weight).abs()
    assert float(diff.max()) <= 3 * 2 * 1.2e-3  # Adam moves an element by about lr a step, whatever its gradient
    assert float(diff.mean()) <= (1e-6 if bits == 32 else 2e-4)
    q = qm.Int8Linear.from_linear(head)
    x = torch.randn(1, 96, device=DEV, generator=g)
    with torch.no_grad():
        y, want = q(x), head(x)
    bound = (x.abs().amax() / 254 * head.weight.abs().sum(1) + x.abs().sum() * head.weight.abs().amax(1) / 254) * 1.01
    assert bool(((y - want).abs()[0] <= bound + 1e-6).all())
    y2 = torch.ops.rpfq.linear_int8(x, q.weight_codes, q.weight_scale, q.bias)
    assert torch.equal(y2, y)


@pytest.mark.gpu
def test_captured_training_step():
    """Loss, gradients and step in one graph, replayed on new data, beside the
    same steps run eagerly."""
    import quant_models as qm
    from quant_models import ops

    g = torch.Generator(device=DEV).manual_seed(4)
    w0, b0 = torch.randn(300, 64, device=DEV, generator=g) * 0.1, torch.zeros(300, device=DEV)
    x, t = torch.zeros(80, 64, device=DEV), torch.zeros(80, dtype=torch.int64, device=DEV)

    def setup():
        w, b = nn.Parameter(w0.clone()), nn.Parameter(b0.clone())
        opt = qm.AdamW([w, b], lr=1e-2)

        def step():
            loss = ops.linear_cross_entropy(x, w, t, b)
            w.grad, b.grad = torch.autograd.grad(loss, [w, b])
            opt.step()
            return loss.detach()

        return w, b, step

    w1, b1, step1 = setup()
    w2, b2, step2 = setup()
    data = [(torch.randn(80, 64, device=DEV, generator=g), torch.randint(0, 300, (80,), device=DEV, generator=g)) for _ in range(6)]

    def feed(k):
        x.copy_(data[k][0])
        t.copy_(data[k][1])

    side = torch.cuda.Stream()
    feed(0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step1()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step1()
    step2()
    for k in range(1, 6):
        feed(k)
        graph.replay()
        got = loss.clone()
        want = step2()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(w1, w2) and torch.equal(b1, b2)


def test_optimizer_groups_and_foreign_states_on_the_host():
    import quant_models as qm

    p, q = nn.Parameter(torch.zeros(4)), nn.Parameter(torch.zeros(4))
    opt = qm.AdamW([p])
    with pytest.raises(ValueError, match="state_bits"):
        opt.add_param_group({"params": [q], "state_bits": 4})
    for kw in ({"amsgrad": True}, {"maximize": True}):
        with pytest.raises(ValueError, match="amsgrad"):
            opt.load_state_dict(torch.optim.AdamW([p], **kw).state_dict())


@pytest.mark.gpu
def test_optimizer_continues_a_torch_run():
    """States that torch.optim.AdamW saved after two steps, then two steps on
    either side (bounds as in test_optimizer_follows_torch)."""
    import quant_models as qm

    a, b, g = _pair(32)
    theirs = torch.optim.AdamW(b, lr=1e-3)
    grads = [[torch.randn(p.shape, device=DEV, generator=g) for p in a] for _ in range(4)]

    def go(params, opt, gs):
        for grad in gs:
            for p, x in zip(params, grad):
                p.grad = x.clone()
            opt.step()

    go(b, theirs, grads[:2])
    mine = qm.AdamW(a, lr=5.0, state_bits=8)
    mine.load_state_dict(theirs.state_dict())
    with torch.no_grad():
        for p, q in zip(a, b):
            p.copy_(q)
    go(a, mine, grads[2:])
    go(b, theirs, grads[2:])
    for p, q in zip(a, b):
        assert float((p - q).abs().max()) <= 2 * 8 * 2.0 ** -24 * (float(q.abs().max()) + 1e-3)
        assert float(mine.state[p]["step"]) == 4 and mine.state[p]["exp_avg"].dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_after_loading_counts_on(bits):
    """Two groups whose counts are equal when they are loaded: each counts for
    itself from then on, so that nothing of a captured step starts over."""
    import quant_models as qm

    a, b, g = _pair(bits)
    groups = lambda p: [{"params": p[:2], "lr": 3e-3}, {"params": p[2:]}]  # noqa: E731
    first = qm.AdamW(groups(a), state_bits=bits)
    for p, q in zip(a, b):
        p.grad = torch.randn(p.shape, device=DEV, generator=g)
        q.grad = torch.empty_like(q).copy_(p.grad)
    first.step()
    saved = copy.deepcopy(first.state_dict())
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    again = qm.AdamW(groups(b), state_bits=bits)
    again.load_state_dict(saved)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again.step()
    for _ in range(3):
        graph.replay()
        first.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q) and float(first.state[p]["step"]) == float(again.state[q]["step"])


@pytest.mark.gpu
def test_captured_steps_that_would_start_over_are_refused():
    import quant_models as qm

    a, _, g = _pair(32)
    for p in a:
        p.grad = torch.randn(p.shape, device=DEV, generator=g)
    opt = qm.AdamW(a)
    before = [p.detach().clone() for p in a]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="states must exist"):
        with torch.cuda.graph(graph):
            opt.step()
    opt.state.clear()
    opt.step()
    assert all(not torch.equal(p, q) for p, q in zip(a, before))
    a[0].grad = None
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="the step before"):
        with torch.cuda.graph(graph):
            opt.step()
    opt.step()
    opt.step()  # the four that step have a count of their own now
    assert [float(opt.state[p]["step"]) for p in a] == [1.0, 3.0, 3.0, 3.0, 3.0]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(8,), (2, 4)])
def test_captured_backward_beside_an_eager_graph_is_refused(shape):
    """The eager graph has bound the leaves to the default stream."""
    from quant_models import ops

    x = torch.randn(*shape, 16, device=DEV)
    w = nn.Parameter(torch.randn(40, 16, device=DEV))
    t = torch.randint(0, 40, shape, device=DEV)
    alive = ops.linear_cross_entropy(x, w, t)
    ops.linear_cross_entropy(x, w, t).backward()  # eagerly there is nothing against it
    w.grad.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            ops.linear_cross_entropy(x, w, t).backward()
    alive.backward()
    assert float(w.grad.abs().max()) > 0
