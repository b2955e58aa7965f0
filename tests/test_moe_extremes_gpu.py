"""Layers of experts whose tokens, or activations, come near the largest number of fp32: the power of two that a row is scaled by is no reason to overflow."""
import pytest
import torch

import miori_b200 as mb
from test_moe_activation_bits_gpu import one_hot

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("bits,group", [(4, 64), (4, 32), (8, 128)])
@pytest.mark.parametrize("exponent", [-100, -60, 0, 60, 117, 118, 119, 124, 127])
@pytest.mark.parametrize("T", [1, 6])
def test_numbers_near_the_largest(bits, group, exponent, T):
    """g[f] = x[f] / 2, u[f] = x[f + 1] / size, h about size / 2, an output h[i] / 2: one weight in a row, all of them powers of two.  silu is rounded three times and u's product once, the
    pair of fp16 is within 2^-22, its sum and the weight's product 2^-24 each: 2^-21, and 2^-35 of a row's largest."""
    N, size = 128, 2.0 ** exponent
    eye = torch.eye(N, device=DEV)
    up, down = one_hot(bits, group, torch.cat((eye, eye.roll(1, 1)))[None]), one_hot(bits, group, eye[None])
    up[1][:, N if bits == 4 else 1:] = 1 / size  # the scales of u's rows
    g = torch.Generator(device=DEV).manual_seed(T)
    x = ((1 + 0.375 * torch.rand(T, N, generator=g, device=DEV)) * size).to(torch.bfloat16)
    x[:, 5::9] *= -1
    router = torch.zeros(1, N, dtype=torch.bfloat16, device=DEV)
    args = (x, router, *up, *down, 1, mb.moe_workspace(T, 1, N, DEV))
    got = mb.moe4(*args, group=group, factor=2.0, flags=mb.MOE_SIGMOID) if bits == 4 else mb.moe_fp8(*args, factor=2.0, flags=mb.MOE_SIGMOID)
    gate = x.double() / 2
    h = gate / (1 + torch.exp(-gate)) * (x.double().roll(-1, 1) / size)
    assert float(h.abs().max()) < 2.0 ** 128
    assert bool(((got.double() - h / 2).abs() <= h.abs() * 2.0 ** -21 + h.abs().amax(1, keepdim=True) * 2.0 ** -35).all()), got
    assert mb.lib.miori_device_error_poll() == 0
