"""classifier_loss where the model is not in training, and what it refuses."""
import pytest
import torch
import torch.nn.functional as F
from test_training_operators import _model

DEV = "cuda"
NAMES = ["rpfq_vit_tiny_patch16_224_q", "rpfq_deit_tiny_patch16_224_q", "rpfq_swin_tiny_patch4_window7_224_q"]


def _labels():
    return torch.tensor([1, 9, -100, 0, 3, 3], device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [False, True])
def test_eval_loss_is_the_models_loss(name, grad):
    """The packed head (no gradient recorded) takes its rows as fp16 under a
    scale each, 2^-11 of a feature: a logit is off by 2^-11 |x| |w| (2-norms), the
    loss by twice that.  Behind the final LayerNorm |x| is sqrt(D) at most, half
    as much again where it is fake-quantized.  The rest is float32."""
    import quant_models as qm

    m = _model(name).eval()
    heads = [h for n, h in m.named_modules() if n.startswith("head") and hasattr(h, "quantized_weight")]
    assert heads
    with torch.no_grad():
        off = max(float(h.quantized_weight().norm(dim=1).max()) * 1.5 * h.in_features ** 0.5 for h in heads) * 2.0 ** -10
    x = torch.randn(6, 3, 32, 32, device=DEV)
    with torch.set_grad_enabled(grad):
        a = qm.classifier_loss(m, x, _labels(), label_smoothing=0.1)
        b = F.cross_entropy(m(x), _labels(), label_smoothing=0.1)
    assert a.requires_grad == b.requires_grad == grad
    assert abs(float(a.detach()) - float(b.detach())) <= 1e-5 * (1 + float(b.detach())) + (0 if grad else off)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_supplied_codes_are_refused_in_eval(name):
    """With supplied codes the head of a model in eval does not run from its
    weight: the loss of that weight would be another one.  In training it does."""
    import quant_models as qm
    from quant_models.inference import load_synthetic_codes

    m = _model(name)
    load_synthetic_codes(m, 5)
    x = torch.randn(6, 3, 32, 32, device=DEV)
    m.train()
    with torch.no_grad():
        a, b = qm.classifier_loss(m, x, _labels()), F.cross_entropy(m(x), _labels())
    assert abs(float(a) - float(b)) <= 1e-5 * (1 + float(b))
    m.eval()
    for grad in (False, True):
        with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="supplied codes"):
            qm.classifier_loss(m, x, _labels())


@pytest.mark.parametrize("name", NAMES)
def test_hooks_are_refused(name):
    """On the host: before anything is computed."""
    import quant_models as qm

    m = _model(name, device="cpu")
    x, t = torch.randn(2, 3, 32, 32), torch.tensor([1, 2])
    head = m.head.fc if "swin" in name else m.head
    for module in (m, m.head, head):
        for add in (module.register_forward_hook, module.register_forward_pre_hook, module.register_full_backward_hook):
            handle = add(lambda *a: None)
            with pytest.raises(ValueError, match="hooks"):
                qm.classifier_loss(m, x, t)
            handle.remove()
    with pytest.raises(TypeError):
        qm.classifier_loss(torch.nn.Sequential(m), x, t)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_eval_loss_of_a_prepared_model(name):
    """fp16 inference: the model rounds its logits and their loss to 2^-11, this
    one the head's weight to 2^-11; both meet the same fp16 features."""
    import quant_models as qm
    from quant_models.inference import prepare_inference

    m = _model(name)
    heads = [h for n, h in m.named_modules() if n.startswith("head") and hasattr(h, "quantized_weight")]
    with torch.no_grad():
        off = max(float(h.quantized_weight().norm(dim=1).max()) * 1.5 * h.in_features ** 0.5 for h in heads)
    prepare_inference(m, DEV, torch.float16)
    x = torch.randn(6, 3, 32, 32, device=DEV, dtype=torch.float16)
    with torch.no_grad():
        z = m(x)
        a, b = qm.classifier_loss(m, x, _labels()), F.cross_entropy(z, _labels())
    # a logit: the weight's rounding and the packed rows', each 2^-11 |x| |w|, and
    # its own; the loss: twice that, and its own rounding
    bound = 2 * (2 * 2.0 ** -11 * off + 2.0 ** -11 * float(z.abs().max())) + 2.0 ** -11 * float(b)
    assert abs(float(a) - float(b)) <= bound
