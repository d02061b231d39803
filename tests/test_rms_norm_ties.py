"""8-bit codes of the norm next to the middle of two: 127 h w / max|h w| of float32
operands, decided as whole numbers decide it."""
import pytest
import torch

DEV = "cuda"
# the largest product's factors, another's, and its code: 254 h w and (2 c + 1) max|h w|
# differ by 2 or 4 of about 2^55, which 53 bits round to a tie
CLOSE = [(16915322, 14822395, 12319022, 13221254, 83), (16944866, 15985151, 14666823, 15341491, 105),
         (24489092, 12502807, 15018217, 16614928, 103), (19420220, 9114981, 12204482, 13990168, 123),
         (17320718, 11097041, 7225357, 15186163, 73), (25980486, 15061741, 16283693, 16745923, 89),
         (25978676, 9079223, 11921305, 15501055, 99), (24610596, 11965587, 12775690, 15699440, 87)]


@pytest.fixture(params=["native", "ctypes"])
def host_path(request, monkeypatch):
    if request.param == "ctypes":
        from quant_models import _native

        monkeypatch.setattr(_native, "host", lambda: None)


def test_the_cases_are_what_they_say():
    for a, b, c, d, code in CLOSE:
        mid = next(m for m in (code - 1, code) if abs(254 * c * d - (2 * m + 1) * a * b) <= 4)
        assert (254 * c * d > (2 * mid + 1) * a * b) == (code == mid + 1) and 254 * c * d != (2 * mid + 1) * a * b
        for n in (a, b, c, d):
            assert torch.tensor(float(n), dtype=torch.float32).item() == n


@pytest.mark.gpu
@pytest.mark.parametrize("features", [2, 9, 700, 2500])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -40])
def test_codes_beside_a_middle(scale, features, host_path):
    from quant_models import ops

    for a, b, c, d, code in CLOSE:
        for x in (0, features - 2):
            h, w = torch.zeros(3, features, device=DEV), torch.ones(features, device=DEV)
            h[:, x], h[:, x + 1] = torch.tensor([a, -a, a]), torch.tensor([c, c, -c])
            w[x], w[x + 1] = b * scale, d * scale
            codes, _ = ops.rms_norm_int8(h * scale, w)
            assert codes[:, x].tolist() == [127, -127, 127] and codes[:, x + 1].tolist() == [code, code, -code]
            assert int(codes.count_nonzero()) == 6
