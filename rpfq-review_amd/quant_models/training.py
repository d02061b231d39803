"""Training steps of the quantized classifiers: AdamW over all tensors in a
few launches, with states in 32 or in 8 bits, and the loss of a model's head
without its logits.
"""
from __future__ import annotations

from collections import defaultdict

import torch
import torch.nn as nn

from .quant_i import QATLinearComplexPhase
from .swin_transformer import SwinTransformer
from .vision_transformer import VisionTransformer, VisionTransformerDistilled


# ---------------------------------------------------------------------------
# loss
# ---------------------------------------------------------------------------
def _no_hooks(module: nn.Module) -> None:
    """Hooks of a forward that is not called would be left out, those that form
    a weight (pruning, spectral norm) among them."""
    if module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks:
        raise ValueError(f"classifier_loss does not call {type(module).__name__}.forward, which has hooks")


def head_operands(layer: nn.Module, x: torch.Tensor):
    """(x, weight, bias) whose linear map is layer(x) in training: a
    phase-quantized layer's activations and weight as its training forward
    quantizes them (straight-through gradients), nn.Linear's as they are."""
    _no_hooks(layer)
    if isinstance(layer, QATLinearComplexPhase):
        if layer._override is not None and layer.runs_packed(x):
            raise ValueError("classifier_loss: the head runs from supplied codes, not from its float weight; "
                             "take F.cross_entropy(model(images), labels)")
        return layer.training_operands(x)
    if type(layer) is not nn.Linear:
        raise TypeError(f"classifier_loss takes a linear head, got {type(layer).__name__}")
    return x, layer.weight, layer.bias


def classifier_loss(model: nn.Module, images: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                    label_smoothing: float = 0.0, reduction: str = "mean") -> torch.Tensor:
    """F.cross_entropy(model(images), labels, ...) of a ViT, DeiT or Swin
    model (this package's, phase-quantized or not) without its logits: the
    model's features, then ops.linear_cross_entropy with the head's weight.
    A distilled DeiT's two heads are averaged, as its eval output is; in
    distilled training the model returns two outputs, which this does not
    take.  In eval, where a head runs packed, its weight is quantized as in
    training: the same codes and scales.  A head that runs from supplied codes
    (load_packed) is refused, and so are hooks on the model or its head, whose
    forward is not called, and models wrapped in another module."""
    from . import ops

    _no_hooks(model)
    if isinstance(model, VisionTransformerDistilled):
        if model.distilled_training and model.training:
            raise ValueError("classifier_loss: distilled training has a loss for each head")
        f = model.forward_features(images)
        # (head(a) + head_dist(b)) / 2 as one layer of both weights on [a, b] / 2
        parts = [head_operands(h, v) for h, v in ((model.head, f[:, 0]), (model.head_dist, f[:, 1]))]
        x = torch.cat([p[0] for p in parts], -1) * 0.5
        weight = torch.cat([p[1].to(p[0].dtype) if not torch.is_autocast_enabled("cuda") else p[1] for p in parts], -1)
        biases = [p[2] for p in parts if p[2] is not None]
        bias = sum(biases) * 0.5 if biases else None
    elif isinstance(model, VisionTransformer):
        x, weight, bias = head_operands(model.head, model.forward_head(model.forward_features(images), pre_logits=True))
    elif isinstance(model, SwinTransformer):
        _no_hooks(model.head)
        x, weight, bias = head_operands(model.head.fc, model.forward_features(images).mean(dim=(1, 2)))
    else:
        raise TypeError(f"classifier_loss takes a VisionTransformer or SwinTransformer, got {type(model).__name__}")
    if x.dtype != weight.dtype and not torch.is_autocast_enabled("cuda"):
        weight = weight.to(x.dtype)
    return ops.linear_cross_entropy(x, weight, labels, bias, ignore_index=ignore_index, label_smoothing=label_smoothing,
                                    reduction=reduction)


# ---------------------------------------------------------------------------
# optimizer
# ---------------------------------------------------------------------------
def _flat(t: torch.Tensor, what: str) -> torch.Tensor:
    """t's memory as it lies, for tensors without gaps (any order of dimensions)."""
    if t.is_contiguous():
        return t
    expect = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda p: p[1]):
        if stride != expect:
            raise ValueError(f"AdamW: {what} of shape {tuple(t.shape)} and strides {t.stride()} has gaps or overlaps")
        expect *= size
    return t.as_strided((t.numel(),), (1,))


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Two tensors of one shape have their elements in one order."""
    return all(s == t for n, s, t in zip(a.shape, a.stride(), b.stride()) if n != 1)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's step (decoupled weight decay) on the device kernel
    (ops.adamw): one launch per 60 tensors of a type.  state_bits 32: float32
    moments; 8: codes of 8 bits with one scale per 256 elements, 2.03 bytes an
    element instead of 8.  Parameters on the device, float32, fp16 or bf16
    (moments and update in float32).  lr may be a float32 device tensor of one
    element.  The steps are counted on the device, so step() can be captured
    into a graph once the states exist, for the parameters that the eager step
    before it took; torch.amp.GradScaler's scale and its
    skipped steps are taken on the device too.  state_dict() and
    load_state_dict() keep the states' types.  Moments of 32 bits follow a change
    of their parameter's memory order; with 8 bits it is refused."""

    _step_supports_amp_scaling = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"eps and weight_decay must not be negative, got {eps} and {weight_decay}")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must be within 0 .. 1, got {betas}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def add_param_group(self, param_group) -> None:
        if param_group.get("state_bits", 8) not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {param_group['state_bits']}")
        super().add_param_group(param_group)

    def _new_state(self, p: torch.Tensor, bits: int, call, steps: dict) -> dict:
        # parameters of one call that start together share one count (and so a launch)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the states must exist before a step is captured (take one eagerly)")
        if call not in steps:
            steps[call] = torch.zeros(1, dtype=torch.float32, device=p.device)
        state = {"step": steps[call]}
        if bits == 32:
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        else:
            from . import ops

            blocks = -(-p.numel() // ops.STATE_BLOCK)
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.int8)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.uint8)
            for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                state[name] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        from . import ops

        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        grad_scale, found_inf = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        # calls: parameters that step now, of one group, type and count; users:
        # all parameters of a count
        calls, users, fresh = defaultdict(list), defaultdict(int), {}
        for k, group in enumerate(self.param_groups):
            bits = group["state_bits"]
            for p in group["params"]:
                state, g = self.state.get(p), p.grad
                if g is not None:
                    if g.is_sparse:
                        raise RuntimeError("AdamW does not take sparse gradients")
                    if not p.is_cuda:
                        raise ValueError("AdamW takes device parameters only")
                    if not state:
                        state = self.state[p] = self._new_state(p, bits, (k, p.dtype, p.device), fresh)
                    lies = p.stride()
                    if state["exp_avg"].stride() != lies or state["exp_avg_sq"].stride() != lies:
                        self._follow(p, state, bits)
                    calls[k, p.dtype, id(state["step"])].append((p, state, g))
                if state:
                    users[id(state["step"])] += 1
        for (k, _, count), taken in calls.items():
            step = taken[0][1]["step"]
            if len(taken) < users[count]:  # a count belongs to one call: these take a copy
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdamW: a captured step takes the parameters that the step before it took")
                users[count] -= len(taken)
                step = step.clone()
                for _, state, _ in taken:
                    state["step"] = step
            self._launch(ops, taken, step, self.param_groups[k], grad_scale, found_inf)
        return loss

    def _launch(self, ops, taken, step, group, grad_scale, found_inf):
        lists = defaultdict(list)
        for p, state, g in taken:
            if g.stride() != p.stride():
                g = torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device=p.device).copy_(g)
            lists["params"].append(_flat(p, "a parameter"))
            lists["grads"].append(_flat(g, "a gradient"))
            lists["exp_avgs"].append(_flat(state["exp_avg"], "a state"))
            lists["exp_avg_sqs"].append(_flat(state["exp_avg_sq"], "a state"))
            if group["state_bits"] == 8:
                lists["exp_avg_scales"].append(state["exp_avg_scale"])
                lists["exp_avg_sq_scales"].append(state["exp_avg_sq_scale"])
        device = step.device
        there = [None if t is None else t.to(device=device, dtype=torch.float32) for t in (grad_scale, found_inf)]
        ops.adamw(step=step, lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                  grad_scale=there[0], found_inf=there[1], **lists)

    @staticmethod
    def _follow(p, state, bits):
        """Lays the moments out as p, whose memory order may have changed since
        (model.to(memory_format=...))."""
        moved = [k for k in ("exp_avg", "exp_avg_sq") if not _same_order(state[k], p)]
        if not moved:
            return
        _flat(p, "a parameter")  # gaps are another matter
        if bits == 8:
            raise ValueError("AdamW: a parameter's memory order is not the one its 8-bit state was made in, whose blocks follow it")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a parameter's memory order has changed: take a step eagerly before one is captured")
        for k in moved:
            state[k] = torch.empty_strided(p.shape, p.stride(), dtype=state[k].dtype, device=p.device).copy_(state[k])

    def state_values(self, p: torch.Tensor):
        """(first, second) moment of a parameter as float32 tensors."""
        from . import ops

        state = self.state[p]
        if "exp_avg_scale" not in state:
            return state["exp_avg"], state["exp_avg_sq"]
        flat = [_flat(state[k], "a state").reshape(-1) for k in ("exp_avg", "exp_avg_sq")]
        values = ops.adamw_state_values(flat, [state["exp_avg_scale"], state["exp_avg_sq_scale"]])
        return tuple(v.as_strided(p.shape, state[k].stride()) for v, k in zip(values, ("exp_avg", "exp_avg_sq")))

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but the states keep their types (codes stay codes,
        moments are float32), and parameters of one group, type and count share
        it again.  Takes what torch.optim.AdamW saved (its moments of fp16 and
        bf16 parameters, kept in their type, as float32), but for its amsgrad and
        maximize."""
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("AdamW has neither amsgrad nor maximize")
        saved = [(i, g.get("state_bits", 32)) for g in state_dict["param_groups"] for i in g["params"]]
        for (i, bits), p in zip(saved, (p for g in self.param_groups for p in g["params"])):
            codes = state_dict["state"].get(i, {}).get("exp_avg")
            if bits == 8 and codes is not None and codes.shape == p.shape and not _same_order(codes, p):
                raise ValueError("AdamW: an 8-bit state was saved of a parameter in another memory order, which its blocks follow")
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            group.setdefault("state_bits", 32)
        params = [(k, p) for k, g in enumerate(self.param_groups) for p in g["params"]]
        counts = {}
        for (i, _), (k, p) in zip(saved, params):
            source = state_dict["state"].get(i)
            if not source:
                continue
            for name, value in source.items():
                if name == "step":
                    at = float(value)
                    call = (k, p.dtype, p.device, at)
                    if call not in counts:
                        counts[call] = torch.full((1,), at, dtype=torch.float32, device=p.device)
                    value = counts[call]
                elif isinstance(value, torch.Tensor):
                    if self.param_groups[k]["state_bits"] == 32:
                        value = value.float()
                    moved = value.to(p.device)
                    value = torch.empty_strided(p.shape, p.stride(), dtype=value.dtype, device=p.device).copy_(moved) \
                        if value.shape == p.shape and name in ("exp_avg", "exp_avg_sq") else moved.clone()
                self.state[p][name] = value
