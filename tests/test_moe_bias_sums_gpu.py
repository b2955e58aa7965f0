"""What the biases of packed weights multiply: a group's sum of activations, which fp32 holds.

The layers have codes of zero and biases of one, or of powers of two, and activations that are powers of two, one of each row 2^22 times others, whose sums take up to 24 bits: fp32 has no
rounding anywhere.  (As products with 2^-24, the least of fp16, a group's sum lost what was 2^-20 of its largest or less.)  What stands between the products is a pair of fp16, all 22 bits of it where it is no
less than 2^-13 of its row's largest, and within 2^-35 of that anyway."""
import pytest
import torch

import miori_b200 as mb
from test_moe_activation_bits_gpu import one_hot

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
N = 256


def layer(x, up, down, group):
    T = x.shape[0]
    router = torch.zeros(1, N, dtype=torch.bfloat16, device=DEV)  # a score of one half, times the factor
    return mb.moe4(x, router, *up, *down, 1, mb.moe_workspace(T, 1, N, DEV), group=group, factor=2.0, flags=mb.MOE_SIGMOID).double()


@pytest.mark.parametrize("group", [64, 32])
@pytest.mark.parametrize("T", [1, 3, 7, 32])
def test_sums_in_front_of_the_first_product(T, group):
    g = torch.Generator(device=DEV).manual_seed(T)
    eye = torch.eye(N, device=DEV)
    up = [t.clone() for t in one_hot(4, group, torch.cat((eye, eye.roll(1, 1)))[None])]
    up[0][:, :N], up[2][:, :N] = 0, 1.0  # g[f]: the sum of x, for every f; u[f] = x[f + 1] / 2
    x = torch.exp2(torch.floor(9 * torch.rand(T, N, generator=g, device=DEV))) * torch.where(torch.rand(T, N, generator=g, device=DEV) < 0.5, -1, 1)  # 2^0 .. 2^8
    x[:, 17] = 2.0 ** 22
    s = x.double().sum(1, keepdim=True)
    assert float(s.min()) > 64 and float(s.max()) < 2 ** 23  # silu(s) is s
    got = layer(x.to(torch.bfloat16), up, one_hot(4, group, eye[None]), group)
    want = s * x.roll(-1, 1) / 4
    assert bool(((got - want).abs() <= want.abs().amax(1, keepdim=True) * 2.0 ** -35).all()), float(((got - want).abs() / want.abs()).max())


@pytest.mark.parametrize("group", [64, 32])
@pytest.mark.parametrize("T", [1, 3, 7, 32])
def test_sums_in_front_of_the_second_product(T, group):
    g = torch.Generator(device=DEV).manual_seed(10 + T)
    eye = torch.eye(N, device=DEV)
    up = [t.clone() for t in one_hot(4, group, torch.cat((eye, eye))[None])]
    up[1][:, :N] = 2.0 ** 8  # g[f] = 2^8 x[f], u[f] = x[f] / 2: h[f] = 2^7 x[f]^2
    x = torch.exp2(torch.floor(5 * torch.rand(T, N, generator=g, device=DEV)))  # 2^0 .. 2^4
    x[:, 5] = 2.0 ** 11
    h = 2 ** 7 * x.double() ** 2  # 2^7 .. 2^15, and one of 2^29
    down = list(one_hot(4, group, torch.zeros(1, N, N, device=DEV)))
    down[2] = torch.exp2(torch.arange(N, device=DEV) % 5 - 2.0)[None, :, None].expand(1, N, N // group).to(torch.bfloat16).contiguous()
    assert float(h.sum(1).max()) < 2 ** 30
    got = layer(x.to(torch.bfloat16), up, down, group)
    assert torch.equal(got, h.sum(1, keepdim=True) * down[2][0, :, 0].double())
