"""Scores of any size that fp32 holds: the largest takes all, and the result is its value exactly.

q is a power of two in every dimension and the keys are constant, distinct bf16 numbers, so scores are exact in fp32 and two of them are
2^-8 of themselves apart at least: beside the largest, each other weight is below 2^-100."""
import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def workspace():
    return mb.attention_workspace(DEV)


def keys(g, L, G, D, sign):
    """Constant, distinct keys between 1 and 2^13, in some order of its own for each head; with sign = 0 every other one negative."""
    bits = torch.arange(L, device=DEV) + 0x3F80  # consecutive bf16 numbers from 1 on
    x = torch.stack([bits[torch.randperm(L, generator=g, device=DEV)] for _ in range(G)], 1).to(torch.int16).view(torch.bfloat16)
    if sign == 0:
        x = torch.where((torch.arange(L, device=DEV) % 2 == 0)[:, None], x, -x)
    return (x if sign >= 0 else -x)[:, :, None].expand(L, G, D).contiguous()


def largest(k, v, n, H):
    """For the last n tokens of a request: the value of the largest key that each of them sees."""
    L, G, _ = k.shape
    top = k[:, :, 0].float().cummax(0).indices[L - n:]  # [n][G]
    return torch.stack([v[top[:, h // (H // G)], h // (H // G)] for h in range(H)], 1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sign", [1, -1, 0])
@pytest.mark.parametrize("power", [12, 20, 26, 40, 90])
@pytest.mark.parametrize("T", [300, 1500])
@pytest.mark.parametrize("shared", [True, False])
def test_prompts(D, sign, power, T, shared, workspace):
    g = torch.Generator(device=DEV).manual_seed(1)
    H, G = 4, 2
    q = torch.full((T, H, D), 2.0 ** power, device=DEV).to(torch.bfloat16)
    k, v = keys(g, T, G, D, sign), torch.randn(T, G, D, generator=g, device=DEV).to(torch.bfloat16)
    out = mb.attention_prompt(q, k, v, torch.tensor([0, T], dtype=torch.int32, device=DEV), workspace=workspace if shared else None)
    torch.cuda.synchronize()
    assert mb.lib.miori_device_error_poll() == 0
    assert torch.equal(out, largest(k, v, T, H))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sign", [1, -1, 0])
@pytest.mark.parametrize("power", [12, 26, 40, 90])
@pytest.mark.parametrize("new", [1, 4, 70])
def test_pages(D, sign, power, new, workspace):
    g = torch.Generator(device=DEV).manual_seed(2)
    H, G, L, page = 4, 2, 1600, 16
    q = torch.full((new, H, D), 2.0 ** power, device=DEV).to(torch.bfloat16)
    k, v = keys(g, L, G, D, sign), torch.randn(L, G, D, generator=g, device=DEV).to(torch.bfloat16)
    pages = [t.view(L // page, page, G, D).transpose(1, 2) for t in (k, v)]
    table, lens = torch.arange(L // page, dtype=torch.int32, device=DEV)[None], torch.tensor([L], dtype=torch.int32, device=DEV)
    out = mb.attention_paged(q, *pages, table, lens, torch.tensor([0, new], dtype=torch.int32, device=DEV), new, workspace=workspace)
    torch.cuda.synchronize()
    assert mb.lib.miori_device_error_poll() == 0
    assert torch.equal(out, largest(k, v, new, H))
