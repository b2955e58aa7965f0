"""Scores that are not numbers.  A softmax over a logit that is none has no numbers at all: the token's row is none either, shares or not, whoever was chosen.  A sigmoid's
is one expert's, which comes last."""
import pytest
import torch

import miori_b200 as mb
import test_moe_gpu as moe

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 128)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("norm", [0, mb.MOE_NORM])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_softmax_of_no_numbers(bits, group, bias, norm, value):
    x, router, ws, b = moe.make(bits, group, 4, 8, 256, 256, 31, bias=bias)
    x[:, 0] = 1.0
    x[2, 0] = 0.0  # NaN * 0 is NaN, and so is infinity * 0
    clean = moe.run(x, router, ws, bits, group, 2, b, norm)
    assert bool(torch.isfinite(clean).all())
    router[6, 0] = value
    got = moe.run(x, router, ws, bits, group, 2, b, norm)
    p = torch.softmax(x.float() @ router.float().T, 1)
    assert bool(torch.isnan(p).all())
    assert bool(torch.isnan(got).all())
    assert mb.lib.miori_device_error_poll() == 0


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 128)])
@pytest.mark.parametrize("norm", [0, mb.MOE_NORM])
def test_a_sigmoid_of_no_number_comes_last(bits, group, norm):
    x, router, ws, _ = moe.make(bits, group, 5, 8, 256, 256, 32)
    zeros = torch.zeros(8, device=DEV)
    out = zeros.clone()
    out[3] = -float("inf")
    want = moe.run(x, router, ws, bits, group, 3, out, norm | mb.MOE_SIGMOID)
    router[3, 0] = float("nan")
    for bias in (None, zeros):
        assert torch.equal(moe.run(x, router, ws, bits, group, 3, bias, norm | mb.MOE_SIGMOID), want)
    # last, and chosen where all are
    assert bool(torch.isnan(moe.run(x, router, ws, bits, group, 8, zeros, norm | mb.MOE_SIGMOID)).all())


@pytest.mark.parametrize("norm", [0, mb.MOE_NORM])
@pytest.mark.parametrize("sigmoid", [0, mb.MOE_SIGMOID])
def test_logits_of_minus_infinity_are_scores_of_zero(norm, sigmoid):
    x, router, ws, _ = moe.make(4, 64, 3, 8, 256, 256, 33)
    x[:, 0] = 1.0
    router[5, 0] = -float("inf")
    lists = moe.choice(x, router, 3, None, bool(sigmoid), bool(norm), 1.0)
    assert all(e != 5 for row in lists for e, _ in row)
    moe.check(x, router, ws, 4, 64, 3, None, norm | sigmoid)
