"""The quantizer's codes where a value is a zero: e4m3(x / s) keeps the sign of a zero quotient."""
import pytest
import torch

from sfnx_amd import moe
from tests.f8_util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", sorted(OUT))
@pytest.mark.parametrize("amax", [0.0, 1.0, 3e4])
def test_quantize_keeps_the_sign_of_zero(amax, t):
    """zeros of both signs, alone in their blocks and beside other values, and quotients that round to zero"""
    x = torch.zeros((3, 272))
    x[:, 1::2] = -0.0
    x[1, 5::7] = amax
    x[2, 0], x[2, 130], x[2, 262] = -amax, amax, amax
    x[2, 3::8], x[2, 4::8] = -amax * 2.0 ** -21, amax * 2.0 ** -21   # 448 2^-21 of a scale: below half the smallest code
    x = x.to(OUT[t])
    q, s = torch.empty((3, 272), dtype=torch.uint8, device="cuda"), torch.empty((3, 3), device="cuda")
    moe.quantize_f8(x.cuda(), q, s)
    wq, ws = quantize(x)
    assert (wq.view(torch.uint8) == 0x80).any()
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu(), wq.view(torch.uint8))
