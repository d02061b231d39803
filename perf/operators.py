"""Operators around the quantized layers, as cases to time and to compare: the
int8 product with scales for each token and channel, the classifier's cross
entropy with its gradient, and the AdamW step.

Each has a plain form (elementary torch operations) and the framework's call.
"""
import math
import os
import sys

import torch

#: False: the plain forms; True: the framework's entry points.
own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
DEV = "cuda"
IGNORE = -100  # target of a row that counts nowhere
BLOCK = 256  # elements that share the scales of an 8-bit optimizer state
HYPER = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.05}


def _ops():
    path = os.path.join(os.getcwd(), "rpfq-review_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from quant_models import ops

    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the classifier of one image: a single token, where latency counts
        {"name": "int8_one_row", "kind": "int8", "rows": 1, "inf": 768, "outf": 1000, "dtype": "fp16", "bias": True},
        # sizes that fit no tile, float32 in and out
        {"name": "int8_odd_f32", "kind": "int8", "rows": 777, "inf": 515, "outf": 333, "dtype": "fp32", "bias": True},
        # qkv of ViT-B/16 for 8 images in bf16
        {"name": "int8_qkv_bf16", "kind": "int8", "rows": 8 * 197, "inf": 768, "outf": 2304, "dtype": "bf16",
         "bias": True},
        # fc1 of ViT-L/16 for 256 images: throughput serving
        {"name": "int8_vit_l_fc1", "kind": "int8", "rows": 256 * 197, "inf": 1024, "outf": 4096, "dtype": "fp16",
         "bias": True},
        # the training batch of a ViT-B/16 with 1000 labels
        {"name": "loss_1000", "kind": "loss", "rows": 64, "classes": 1000, "inf": 768, "dtype": "bf16", "bias": True,
         "smooth": 0.1, "ignored": 0.0, "train": True},
        # float32 training over a label set of odd sizes, some rows unlabelled
        {"name": "loss_odd_f32", "kind": "loss", "rows": 333, "classes": 10007, "inf": 385, "dtype": "fp32",
         "bias": True, "smooth": 0.1, "ignored": 0.2, "train": True},
        # fp16 (autocast) training over 20,000 labels
        {"name": "loss_20000_fp16", "kind": "loss", "rows": 2048, "classes": 20000, "inf": 1024, "dtype": "fp16",
         "bias": False, "smooth": 0.0, "ignored": 0.1, "train": True},
        # the largest: every token of many sequences against a large vocabulary
        {"name": "loss_65536", "kind": "loss", "rows": 8192, "classes": 65536, "inf": 768, "dtype": "bf16",
         "bias": False, "smooth": 0.0, "ignored": 0.0, "train": True},
        # validation over a large vocabulary: the loss of each row, no gradient
        {"name": "loss_131072_eval", "kind": "loss", "rows": 500, "classes": 131072, "inf": 1024, "dtype": "bf16",
         "bias": False, "smooth": 0.0, "ignored": 0.0, "train": False},
        # only the head is tuned: two small tensors, where latency counts
        {"name": "adamw_head", "kind": "adamw", "layout": "head", "dim": 768, "depth": 0, "classes": 1000,
         "dtype": "fp32", "bits": 32},
        # a ViT-B/16 in float32 with float32 states
        {"name": "adamw_vit_b", "kind": "adamw", "layout": "vit", "dim": 768, "depth": 12, "classes": 1000,
         "dtype": "fp32", "bits": 32},
        # a ViT-L/16 with states in 8 bits
        {"name": "adamw_vit_l_8bit", "kind": "adamw", "layout": "vit", "dim": 1024, "depth": 24, "classes": 1000,
         "dtype": "fp32", "bits": 8},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _features(rng):
    """A layer's width: one of the model family's, or any."""
    return rng.choice([96, 192, 384, 768, 1024, 1536, 4096]) if rng.random() < 0.5 else _log_int(rng, 33, 4096)


def draw(rng):
    kind = rng.choice(["int8", "loss", "adamw"])
    if kind == "int8":
        case = {"kind": kind, "inf": _features(rng), "outf": _log_int(rng, 16, 8192),
                "dtype": rng.choice(["fp16", "bf16", "fp32"]), "bias": rng.random() < 0.7}
        most = 50432 * 1024 * 4096 / (case["inf"] * case["outf"])
        case["rows"] = _log_int(rng, 1, max(1, min(65536, int(most))))
        return case
    if kind == "loss":
        case = {"kind": kind, "classes": _log_int(rng, 100, 131072), "inf": min(1024, _features(rng)),
                "dtype": rng.choice(["fp16", "bf16", "bf16", "fp32"]), "bias": rng.random() < 0.5,
                "smooth": rng.choice([0.0, 0.0, 0.1]), "ignored": rng.choice([0.0, 0.3]),
                "train": rng.random() < 0.75}
        most = 0.3 * 8192 * 65536 * 768 / (case["classes"] * case["inf"])
        case["rows"] = _log_int(rng, 1, max(1, min(16384, int(most))))
        return case
    dim = rng.choice([96, 192, 384, 768, 1024])
    return {"kind": kind, "layout": rng.choice(["head", "vit", "ragged"]), "dim": dim,
            "depth": rng.randrange(1, 25 if dim < 1024 else 13), "classes": _log_int(rng, 10, 20000),
            "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "bits": rng.choice([8, 32])}


def _sizes(case):
    """Elements of each parameter tensor of an optimizer case."""
    d, depth, classes = case["dim"], case["depth"], case["classes"]
    head = [classes * d, classes]
    if case["layout"] == "head":
        return head
    if case["layout"] == "ragged":  # odd sizes of many magnitudes
        return head + [1 + (7919 * (i + 1) * d) % (64 * d + 13 * i) for i in range(6 * depth)]
    block = [d, d, 3 * d * d, 3 * d, d * d, d, d, d, 4 * d * d, 4 * d, 4 * d * d, d]
    return [d, 197 * d, 768 * d, d] + depth * block + [d, d] + head


def work(case):
    es = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "int8":
        m, k, n = case["rows"], case["inf"], case["outf"]
        return {"bytes": m * k * es + n * k + 4 * n + (4 * n if case["bias"] else 0) + m * n * es, "flops": 2 * m * n * k}
    if case["kind"] == "loss":
        m, k, n = case["rows"], case["inf"], case["classes"]
        ends = (m * k + n * k + (n if case["bias"] else 0)) * es
        if case["train"]:
            return {"bytes": 2 * ends + 8 * m + 4, "flops": 6 * m * n * k}
        return {"bytes": ends + 8 * m + 4 * m, "flops": 2 * m * n * k}
    n = sum(_sizes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (3 * es + state), "flops": 15 * n}


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------
def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _power_of_two(top):
    """The scale of a block of 8-bit states: the power of two at or above its
    largest, 2^-126 at least, 0 for zeros."""
    part, e = torch.frexp(top.double())
    s = torch.ldexp(torch.ones_like(part), torch.where(part == 0.5, e - 1, e)).clamp_min(2.0 ** -126)
    return torch.where(top > 0, s, 0.0).float()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "int8":
        m, k, n = case["rows"], case["inf"], case["outf"]
        weight = _normal(g, n, k, scale=0.02)
        top = weight.abs().amax(1)
        # activations behind a LayerNorm, a few channels larger than the rest
        x = _normal(g, m, k) * (1 + 4 * (torch.rand(k, generator=g, device=DEV) < 0.02))
        return {"case": case, "x": x.to(dt), "codes": torch.round(weight * (127 / top[:, None])).to(torch.int8),
                "scale": top / 127, "bias": _normal(g, n, scale=0.1) if case["bias"] else None}
    if case["kind"] == "loss":
        m, k, n = case["rows"], case["inf"], case["classes"]
        # logits of unit spread to 2; half of the rows are answered well
        weight = _normal(g, n, k, scale=2 / math.sqrt(k))
        target = torch.randint(0, n, (m,), generator=g, device=DEV)
        sure = 3 * (torch.rand(m, 1, generator=g, device=DEV) < 0.5)
        x = _normal(g, m, k) + sure * weight[target]
        target[torch.rand(m, generator=g, device=DEV) < case["ignored"]] = IGNORE
        target[0] = n - 1  # one row at least has a label
        return {"case": case, "x": x.to(dt).requires_grad_(case["train"]),
                "weight": weight.to(dt).requires_grad_(case["train"]), "target": target,
                "bias": _normal(g, n, scale=0.5).to(dt).requires_grad_(case["train"]) if case["bias"] else None}
    # Parameters, gradients and states lie one behind another, each tensor from
    # a block's start on; the list holds each tensor's part of them.
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    total = BLOCK * sum(blocks)
    inside = torch.cat([(torch.arange(b * BLOCK, device=DEV) < n) for n, b in zip(sizes, blocks)])
    flat = {"params": (_normal(g, total, scale=0.02) * inside).to(dt),
            "grads": (_normal(g, total, scale=1e-3) * torch.rand(total, generator=g, device=DEV) * inside).to(dt)}
    m, v = 1e-4 * _normal(g, total) * inside, 1e-7 * torch.rand(total, generator=g, device=DEV).square() * inside
    if case["bits"] == 32:
        flat |= {"exp_avgs": m, "exp_avg_sqs": v}
    else:
        m, v = m.view(-1, BLOCK), v.view(-1, BLOCK)
        sm, sv = _power_of_two(m.abs().amax(1)), _power_of_two(v.amax(1))
        flat |= {"exp_avgs": torch.round(127 * torch.sign(m) * (m.abs() / sm.clamp_min(1e-30)[:, None]).sqrt()).to(torch.int8).view(-1),
                 "exp_avg_sqs": torch.round(255 * (v / sv.clamp_min(1e-30)[:, None]).sqrt().sqrt()).to(torch.uint8).view(-1),
                 "exp_avg_scales": sm, "exp_avg_sq_scales": sv}
    at = [BLOCK * sum(blocks[:i]) for i in range(len(sizes))]
    lists = {k: [t[a:a + n] for a, n in zip(at, sizes)] for k, t in flat.items() if not k.endswith("scales")}
    lists |= {k: [t[a // BLOCK:a // BLOCK + b] for a, b in zip(at, blocks)] for k, t in flat.items() if k.endswith("scales")}
    return {"case": case, "flat": flat, "lists": lists, "step": torch.full((1,), 100.0, device=DEV)}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"int8": _run_int8, "loss": _run_loss, "adamw": _run_adamw}[state["case"]["kind"]](state)


def _run_int8(s):
    if own:
        return _ops().linear_int8(s["x"], s["codes"], s["scale"], s["bias"])
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    codes = torch.round(x.double() * 127 / top.double())  # 64 bits: values next to the middle of two codes
    codes = torch.where(top > 0, codes, 0).float()
    y = codes @ s["codes"].float().t() * (top / 127) * s["scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _run_loss(s):
    case, x, weight, target, bias = s["case"], s["x"], s["weight"], s["target"], s["bias"]
    train, smooth = case["train"], case["smooth"]
    if own:
        loss = _ops().linear_cross_entropy(x, weight, target, bias, ignore_index=IGNORE, label_smoothing=smooth,
                                           reduction="mean" if train else "none")
        if not train:
            return {"loss": loss}
        leaves = [x, weight] + ([bias] if bias is not None else [])
        return {"loss": loss.detach(), "grads": list(torch.autograd.grad(loss, leaves))}
    with torch.no_grad():
        xf, wf = x.float(), weight.float()
        logits = xf @ wf.t()
        if bias is not None:
            logits += bias.float()
        valid = target != IGNORE
        at = torch.where(valid, target, 0)[:, None]
        picked = logits.gather(1, at)[:, 0]
        mean = logits.mean(1) if smooth else 0.0
        top = logits.amax(1, keepdim=True)
        p = logits.sub_(top).exp_()
        total = p.sum(1, keepdim=True)
        lse = (top + total.log())[:, 0]
        rows = torch.where(valid, lse - (1 - smooth) * picked - smooth * mean, 0.0)
        if not train:
            return {"loss": rows}
        count = valid.sum()
        dz = p.div_(total)
        if smooth:
            dz -= smooth / case["classes"]
        dz.scatter_add_(1, at, torch.full_like(at, smooth - 1, dtype=torch.float32))
        dz *= (valid / count)[:, None]
        grads = [(dz @ wf).to(x.dtype), (dz.t() @ xf).to(weight.dtype)]
        if bias is not None:
            grads.append(dz.sum(0).to(bias.dtype))
        return {"loss": rows.sum() / count, "grads": grads}


def _run_adamw(s):
    f, l = s["flat"], s["lists"]
    small = s["case"]["bits"] == 8
    if own:
        ops = _ops()
        ops.adamw(l["params"], l["grads"], l["exp_avgs"], l["exp_avg_sqs"], s["step"],
                  exp_avg_scales=l.get("exp_avg_scales"), exp_avg_sq_scales=l.get("exp_avg_sq_scales"), **HYPER)
        if not small:
            return {"params": f["params"], "exp_avgs": f["exp_avgs"], "exp_avg_sqs": f["exp_avg_sqs"], "step": s["step"]}
        m, v = ops.adamw_state_values([f["exp_avgs"], f["exp_avg_sqs"]], [f["exp_avg_scales"], f["exp_avg_sq_scales"]])
        return {"params": f["params"], "exp_avgs": m, "exp_avg_sqs": v, "step": s["step"]}
    b1, b2 = HYPER["betas"]
    s["step"] += 1
    t = s["step"].double()
    c1, c2 = (1 - b1 ** t).float(), (1 - b2 ** t).sqrt().float()
    p, g = f["params"].float(), f["grads"].float()
    if not small:
        m, v = f["exp_avgs"].mul_(b1).add_(g * (1 - b1)), f["exp_avg_sqs"].mul_(b2).add_(g * g * (1 - b2))
        m1, v1 = m, v
    else:  # 64 bits: values next to the middle of two codes
        gd = g.double().view(-1, BLOCK)
        c = f["exp_avgs"].double().view(-1, BLOCK) / 127
        md = b1 * (c * c.abs() * f["exp_avg_scales"].double()[:, None]) + (1 - b1) * gd
        c = f["exp_avg_sqs"].double().view(-1, BLOCK) / 255
        vd = b2 * (c.square().square() * f["exp_avg_sq_scales"].double()[:, None]) + (1 - b2) * gd * gd
        m1, v1 = md.float().view(-1), vd.float().view(-1)
        sm, sv = _power_of_two(md.abs().amax(1)), _power_of_two(vd.amax(1))
        top = torch.where(sm > 0, sm, 1.0).double()[:, None]
        cm = torch.round(127 * (md.abs() / top).sqrt()).clamp_max(127) * md.sign()
        top = torch.where(sv > 0, sv, 1.0).double()[:, None]
        cv = torch.maximum(torch.round(255 * (vd / top).sqrt().sqrt()).clamp_max(255), (vd > 0).double())
        f["exp_avgs"].copy_(cm.view(-1))
        f["exp_avg_sqs"].copy_(cv.view(-1))
        f["exp_avg_scales"].copy_(sm)
        f["exp_avg_sq_scales"].copy_(sv)
        m = ((cm / 127) * (cm / 127).abs() * sm.double()[:, None]).float().view(-1)
        v = ((cv / 255).square().square() * sv.double()[:, None]).float().view(-1)
    p = p * (1 - HYPER["lr"] * HYPER["weight_decay"]) - HYPER["lr"] * (m1 / c1) / (v1.sqrt() / c2 + HYPER["eps"])
    f["params"].copy_(p)
    return {"params": f["params"], "exp_avgs": m, "exp_avg_sqs": v, "step": s["step"]}


# ---------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"int8": _exact_int8, "loss": _exact_loss, "adamw": _exact_adamw}[case["kind"]](s)


def _exact_int8(s):
    x = s["x"].double()
    top = x.abs().max(dim=1).values
    q = (127 * x / top.clamp_min(1e-300).unsqueeze(1)).round()
    y = torch.einsum("mk,nk->mn", q, s["codes"].double()) * (top / 127).unsqueeze(1) * s["scale"].double().unsqueeze(0)
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_loss(s):
    case = s["case"]
    x, w, n, e = s["x"].double(), s["weight"].double(), case["classes"], case["smooth"]
    z = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].double())
    valid = s["target"].ne(IGNORE)
    # the label distribution that each row is held to
    q = torch.full_like(z, e / n)
    rows = torch.nonzero(valid)[:, 0]
    q[rows, s["target"][rows]] += 1 - e
    logp = torch.log_softmax(z, dim=1)
    each = -(q * logp).sum(dim=1).masked_fill(~valid, 0.0)
    if not case["train"]:
        return {"loss": each}
    dz = (logp.exp() - q).masked_fill(~valid.unsqueeze(1), 0.0) / valid.sum()
    grads = [torch.mm(dz, w), torch.mm(dz.t().contiguous(), x)]
    if s["bias"] is not None:
        grads.append(dz.sum(dim=0))
    return {"loss": each.sum() / valid.sum(), "grads": grads}


def _levels(top, power):
    """The values, relative to the scale, from which on a code is the nearest."""
    return ((torch.arange(top, device=DEV, dtype=torch.float64) + 0.5) / top).pow(power)


def _exact_adamw(s):
    f, (b1, b2) = s["flat"], HYPER["betas"]
    t = float(s["step"]) + 1
    p, g = f["params"].double(), f["grads"].double()
    if s["case"]["bits"] == 32:
        m, v = f["exp_avgs"].double(), f["exp_avg_sqs"].double()
    else:
        c = f["exp_avgs"].double()
        m = c.sign() * (c / 127).pow(2) * f["exp_avg_scales"].double().repeat_interleave(BLOCK)
        v = (f["exp_avg_sqs"].double() / 255).pow(4) * f["exp_avg_sq_scales"].double().repeat_interleave(BLOCK)
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g.square(), v, b2)
    update = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + HYPER["eps"])
    p = p - HYPER["lr"] * (HYPER["weight_decay"] * p + update)
    if s["case"]["bits"] == 8:
        sm = m.abs().view(-1, BLOCK).max(dim=1).values.log2().ceil().exp2().repeat_interleave(BLOCK)
        sv = v.view(-1, BLOCK).max(dim=1).values.log2().ceil().exp2().repeat_interleave(BLOCK)
        c = torch.bucketize(m.abs() / sm.clamp_min(1e-300), _levels(127, 2)).double()
        m = m.sign() * (c / 127).square() * sm
        c = torch.bucketize(v / sv.clamp_min(1e-300), _levels(255, 4)).double()
        v = torch.where((v > 0) & (c == 0), 1.0, c).div(255).pow(4) * sv
    return {"params": p, "exp_avgs": m, "exp_avg_sqs": v, "step": torch.full((1,), t, dtype=torch.float64, device=DEV)}
