"""Values that are not finite, left out of a product and added at its end, over many items of one and of two row tiles."""
import math

import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("lengths", [[60] + [20] * 100, [20] * 12 + [64, 20, 50, 20] * 10, [700] + [30] * 30 + [64] * 3 + [20] * 9 + [200]])
def test_every_prompt_with_a_value_that_is_not_finite(D, shared, lengths):
    """Heads 16 to a key head: a row tile is eight tokens, an item sixteen, so that prompts have items with and without a second row tile.
    Token n - 3 of each prompt has infinities in some dimensions, which reach it and those behind it and nobody else."""
    g = torch.Generator(device=DEV).manual_seed(1)
    H, G, T = 32, 2, sum(lengths)
    lengths = lengths + [600]  # enough tokens for the tensor-memory kernel
    T += 600
    q, k, v = (torch.randn(T, h, D, generator=g, device=DEV).to(torch.bfloat16) for h in (H, G, G))
    cu = torch.tensor([0] + lengths, device=DEV).cumsum(0).to(torch.int32)
    ws = mb.attention_workspace(DEV) if shared else None
    clean = mb.attention_prompt(q, k, v, cu, workspace=ws)
    hit = torch.zeros(T, H, D, dtype=torch.bool, device=DEV)
    for i, (a, n) in enumerate(zip(cu.tolist(), lengths)):
        v[a + n - 3, 1, i % 7::7] = math.inf
        hit[a + n - 3:a + n, H // 2:, i % 7::7] = True
    for _ in range(10):
        got = mb.attention_prompt(q, k, v, cu, workspace=ws)
        assert torch.equal(got[~hit], clean[~hit])
        assert (got[hit] == math.inf).all()
    torch.cuda.synchronize()
    assert mb.lib.miori_device_error_poll() == 0
