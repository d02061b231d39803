"""to_int8 on the host: which layers it replaces, and what a refusal leaves."""
import pytest
import torch
import torch.nn as nn
from test_training_operators import _model


class _Scaled(nn.Linear):
    """A linear layer with a forward of its own."""

    def forward(self, x):
        return 3.0 * super().forward(x)


def test_subclasses_with_their_own_forward_stay():
    from quant_models.inference import to_int8
    from quant_models.int8 import Int8Linear

    torch.manual_seed(0)
    m = nn.ModuleDict({"a": nn.Linear(8, 8), "s": _Scaled(8, 8), "att": nn.MultiheadAttention(8, 2, batch_first=True)}).eval()
    x = torch.randn(2, 3, 8)
    with torch.no_grad():
        s, att = m["s"](x), m["att"](x, x, x)[0]
        assert to_int8(m) == 1 and isinstance(m["a"], Int8Linear)
        assert torch.equal(m["s"](x), s) and torch.equal(m["att"](x, x, x)[0], att)


def test_a_refusal_leaves_the_model_as_it_was():
    from quant_models.inference import load_synthetic_codes, quant_layers, to_int8
    from quant_models.int8 import Int8Linear

    m = _model(device="cpu")
    layers = [layer for _, layer in quant_layers(m)]
    load_synthetic_codes(m, 3)
    last = m.blocks[-1].mlp.fc2  # it alone runs from supplied codes
    for layer in layers:
        if layer is not last:
            layer._override = None
    with pytest.raises(ValueError, match="supplied codes"):
        to_int8(m)
    assert [layer for _, layer in quant_layers(m)] == layers and not any(isinstance(c, Int8Linear) for c in m.modules())
    last._override = None
    assert to_int8(m) >= len(layers)


def test_one_layer_in_two_places_stays_one():
    from quant_models.inference import to_int8
    from quant_models.int8 import Int8Linear

    m = nn.Module()
    m.a = m.b = nn.Linear(8, 8)
    m.inner = nn.Sequential(m.a, nn.Linear(8, 4))
    assert to_int8(m) == 2
    assert isinstance(m.a, Int8Linear) and m.a is m.b and m.a is m.inner[0]
