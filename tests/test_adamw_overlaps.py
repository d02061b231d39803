"""adamw refuses whatever it would write twice or read after it was written."""
import pytest
import test_adamw as base
import torch

DEV = "cuda"
host_path = base.host_path


@pytest.mark.gpu
@pytest.mark.parametrize("names", [("exp_avg_scales", "exp_avg_scales"), ("exp_avg_sq_scales", "exp_avg_sq_scales"),
                                   ("exp_avg_scales", "exp_avg_sq_scales")])
def test_scales_of_two_tensors_in_one_place(names):
    from quant_models import ops

    t = {k: list(v) for k, v in base._tensors(torch.float32, 8, 1, [(300,), (512,)]).items()}
    both = torch.zeros(3, device=DEV)
    t[names[0]][0], t[names[1]][1] = both[:2], both[1:]
    old = [p.clone() for p in t["params"]]
    step = torch.zeros(1, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.adamw(step=step, **t)
    assert float(step) == 0 and all(torch.equal(a, b) for a, b in zip(t["params"], old))
    both = torch.zeros(4, device=DEV)
    t[names[0]][0], t[names[1]][1] = both[:2], both[2:]
    ops.adamw(step=step, **t)
    assert float(step) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_and_step_in_what_is_written(bits):
    from quant_models import ops

    make = lambda: {k: list(v) for k, v in base._tensors(torch.float32, bits, 1, [(8,), (9,)]).items()}  # noqa: E731
    step = torch.zeros(1, device=DEV)
    wide = torch.zeros(16, device=DEV)
    for first, last in ((0, 8), (7, 15), (3, 11)):
        t = make()
        t["params"][0], t["grads"][0] = wide[4:12], wide[first:first + 8]
        with pytest.raises(ValueError, match="overlap"):
            ops.adamw(step=step, **t)
    t = make()
    t["params"][0] = wide[4:12]
    with pytest.raises(ValueError, match="overlap"):
        ops.adamw(step=wide[5:6], **t)
    assert float(step) == 0 and float(wide.abs().max()) == 0
    # neighbours, and two parameters with one gradient, are none of this
    t = make()
    t["params"][0], t["grads"][0] = wide[:8], wide[8:]
    ops.adamw(step=step, **t)
    t = {k: list(v) for k, v in base._tensors(torch.float32, bits, 1, [(8,), (8,)]).items()}
    t["grads"][1] = t["grads"][0]
    ops.adamw(step=step, **t)
    assert float(step) == 2
