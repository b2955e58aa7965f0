"""rope_kv begins beside the launch before it; without LAUNCH_PDL it reads nothing, its weights included, before that one is done."""
import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def chain(D, H, G, T, which, between):
    """Twenty rounds of a launch that writes one of rope_kv's weights and of the rope_kv that reads it."""
    g = torch.Generator(device=DEV).manual_seed(1)
    half = D // 2
    qkv = torch.randn(T, (H + 2 * G) * D, generator=g, device=DEV)
    positions, slots = torch.randint(0, 40000, (3, T), generator=g, device=DEV).to(torch.int32), torch.arange(T, dtype=torch.int32, device=DEV)
    turns, axes = mb.rope_turns(D, theta=1e4, sections=(half - 20, 10, 10), device=DEV)
    gamma, one, table = torch.ones(D, dtype=torch.bfloat16, device=DEV), torch.ones(2 * half, dtype=torch.int32, device=DEV), torch.zeros(2 * half, 64, dtype=torch.int32, device=DEV)
    gammas = [gamma, gamma]
    cache = torch.zeros(2, -(-T // 16), G, 16, D, dtype=torch.bfloat16, device=DEV)
    seen = []
    for i in range(20):
        x = torch.randn(2, D, generator=g, device=DEV)
        held = torch.randint(0, 3 if which == "axes" else 2 ** 29, (2 * half,), generator=g, device=DEV).to(torch.int32)
        torch.cuda.synchronize()
        if which == "gamma":
            gammas = list(mb.rmsnorm(x, gamma, 1e-5))
        else:  # the positions of a step: whole numbers of any kind
            words = mb.page_slots(held, one, table, one, i32([0]), 1 << 24, 2 * half)[1]
            if which == "axes":
                axes = words[:half]
            else:
                turns = words.view(torch.int64)
        between()
        q = mb.rope_kv(qkv, turns, positions, slots, cache[0], cache[1], H, axes=axes, gamma_q=gammas[0], gamma_k=gammas[1], eps=1e-5)
        seen += [q, cache[0].clone()]
    torch.cuda.synchronize()
    return seen


@pytest.mark.parametrize("which", ["gamma", "axes", "turns"])
@pytest.mark.parametrize("D,H,G,T", [(128, 16, 4, 1), (128, 16, 4, 2000), (64, 2, 1, 7)])
def test_weights_of_the_launch_before(which, D, H, G, T):
    want = chain(D, H, G, T, which, torch.cuda.synchronize)
    for _ in range(5):
        got = chain(D, H, G, T, which, lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert mb.lib.miori_device_error_poll() == 0
