"""The activation between a layer's products, silu(g) u, keeps its bits: what is rounded on the way to the second product is a pair of 11 bits each.

Every other operation of these layers is exact: weights are powers of two or zero, one in a row, scores are one half and the factor 2, so an output is one
activation times a power of two.  Tolerance: of the activation itself in fp32, g and u exact, e^-g within 2 units (2^-23 each) of a sum 1 + e^-g that is at least as large, that sum, the
quotient and the product with u rounded once each (2^-24): 7 * 2^-24; of the pair, 2^-11 of 2^-11 of a value, or of values that are small beside their row's
largest 2^-25 times the 16 by which some codes' are taken smaller, of a largest of 2^14 at least: 2^-35 of that; the pair's sum, and the sum of the experts: 2^-24 each.  Rounded to 11 bits
alone, a value would be off by up to 2^-11."""
import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP8 = torch.float8_e4m3fn


def one_hot(bits, group, matrices):
    """Weights whose values are those of `matrices` [E][N][K], ones and zeros, in the layer's format."""
    if bits == 8:
        E, N, K = matrices.shape
        return matrices.to(FP8), torch.full((E, -(-N // 128), -(-K // 128)), 0.5, device=DEV)
    shifts = torch.arange(0, 32, 4, device=DEV)
    words = (matrices.long().unflatten(-1, (-1, 8)) << shifts).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    scales = torch.full((*matrices.shape[:2], matrices.shape[2] // group), 0.5, dtype=torch.bfloat16, device=DEV)
    return words, scales, torch.zeros_like(scales)


@pytest.mark.parametrize("bits,group", [(4, 64), (4, 32), (8, 128)])
@pytest.mark.parametrize("T,E,top", [(1, 4, 2), (3, 1, 1), (4, 3, 1), (5, 1, 1), (6, 4, 3), (8, 2, 2), (13, 20, 3), (32, 1, 1), (32, 8, 4)])
def test_the_activation_keeps_its_bits(bits, group, T, E, top):
    N = 256
    g = torch.Generator(device=DEV).manual_seed(T + E)
    rand = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    # of sizes that bf16 and the activations' scaling hold without a rounding
    x = ((1 + rand(T, N)) * torch.exp2(torch.floor(16 * rand(T, N)) - 8) * torch.where(rand(T, N) < 0.4, -1, 1) * torch.exp2(torch.floor(20 * rand(T, 1)) - 12)).to(torch.bfloat16)
    eye = torch.eye(N, device=DEV)
    turns = [e % 7 for e in range(E)]
    up = torch.stack([torch.cat((eye.roll(n, 1), eye.roll(3 * n + 1, 1))) for n in turns])  # g[f] = x[f + n] / 2, u[f] = x[f + 3 n + 1] / 2
    down = torch.stack([eye.roll(5 * n, 1) for n in turns])                                  # out[i] = h[i + 5 n] / 2
    router = torch.zeros(E, N, dtype=torch.bfloat16, device=DEV)
    ws = one_hot(bits, group, up) + one_hot(bits, group, down)
    workspace = mb.moe_workspace(T, top, N, DEV)
    want, tol = torch.zeros(T, N, dtype=torch.float64, device=DEV), torch.zeros(T, N, dtype=torch.float64, device=DEV)
    # equal scores: the experts of lowest index
    for n in turns[:top]:
        gate, rise = x.double().roll(-n, 1) / 2, x.double().roll(-(3 * n + 1), 1) / 2
        h = gate / (1 + torch.exp(-gate)) * rise
        room = h.abs() * ((8 + top) * 2.0 ** -24 + 2.0 ** -22) + h.abs().amax(1, keepdim=True) * 2.0 ** -35
        want += h.roll(-5 * n, 1) / 2
        tol += room.roll(-5 * n, 1) / 2
    call = (lambda **kw: mb.moe4(x, router, *ws, top, workspace, group=group, factor=2.0, flags=mb.MOE_SIGMOID, **kw)) if bits == 4 else (
        lambda **kw: mb.moe_fp8(x, router, *ws, top, workspace, factor=2.0, flags=mb.MOE_SIGMOID, **kw))
    got = call()
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (float((off / tol).max()), int((off > tol).sum()))
    assert torch.equal(got, call()) and mb.lib.miori_device_error_poll() == 0
