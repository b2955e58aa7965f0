"""The weights of a row add up to one, whatever rounding each of them has gone through.

Values that are the same number c for all keys: the result is c itself.  It is sum(p c) / sum(p) over the same rounded p, so that only
fp32 sums stand between it and c: 2^-24 a term in each, of at most 2^14 terms and 2^3 parts, and 2^-21 for the rescaling of the parts,
below 2^-9 of c together, and bf16 numbers are 2^-8 of c or more apart.  A sum over other p than those of the product
is off by up to 2^-8 of c where one key outweighs the rest.
"""
import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def workspace():
    return mb.attention_workspace(DEV)


def rand(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(torch.bfloat16)


def constants(g, rows, G, D):
    """A number for each key head and dimension, the same for all rows."""
    return rand(g, 1, G, D).expand(rows, G, D).contiguous()


def check(out, v):
    torch.cuda.synchronize()
    assert mb.lib.miori_device_error_poll() == 0
    G, D = v.shape[1:]
    want = v[0].repeat_interleave(out.shape[1] // G, 0).expand_as(out)
    assert torch.equal(out, want), f"{(out != want).sum().item()} of {out.numel()} differ"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[77], [300, 40], [700, 3, 1500], [2500]])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("q_scale", [0.3, 3.0, 6.0])
def test_prompts(D, lengths, shared, q_scale, workspace):
    g = torch.Generator(device=DEV).manual_seed(1)
    H, G, T = 8, 2, sum(lengths)
    cu = torch.tensor([0] + lengths, device=DEV).cumsum(0).to(torch.int32)
    v = constants(g, T, G, D)
    check(mb.attention_prompt(rand(g, T, H, D, scale=q_scale), rand(g, T, G, D), v, cu, workspace=workspace if shared else None), v)


@pytest.mark.parametrize("D,H,G", [(128, 16, 4), (128, 8, 8), (64, 32, 8), (64, 8, 2)])
@pytest.mark.parametrize("new", [1, 3, 5, 70])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("q_scale", [0.3, 3.0, 6.0])
def test_pages(D, H, G, new, shared, q_scale, workspace):
    g = torch.Generator(device=DEV).manual_seed(2)
    page, held = 16, [9000, 5, 250, 1200]
    R, width = len(held), -(-(max(held) + new) // page)
    table = torch.randperm(R * width, generator=g, device=DEV).to(torch.int32).view(R, width)
    k, v = rand(g, R * width, G, page, D), constants(g, R * width, G, D)[:, :, None].expand(-1, -1, page, -1).contiguous()
    lens = torch.tensor([h + new for h in held], dtype=torch.int32, device=DEV)
    cu = torch.arange(0, (R + 1) * new, new, dtype=torch.int32, device=DEV)
    check(mb.attention_paged(rand(g, R * new, H, D, scale=q_scale), k, v, table, lens, cu, new, workspace=workspace if shared else None), v[:, :, 0])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rise", [2.0, 4.0, 5.4, 6.5, 7.5])
def test_one_key_that_outweighs_the_rest_behind_the_first_tile(D, rise, workspace):
    """Scores of unit normals, and of `rise` for key 200 of 256: with a maximum that moves or stands still, in each kernel."""
    g = torch.Generator(device=DEV).manual_seed(3)
    H, G, L, page = 4, 1, 256, 16
    q = rand(g, 1, H, D)
    k = rand(g, L, G, D)
    direction = q[0, 0].float() / q[0, 0].float().square().sum()
    k[200, 0] = (direction * rise * D ** 0.5).to(torch.bfloat16)  # q0 . k = rise * sqrt(D)
    q[0, 1:] = q[0, 0]
    v = constants(g, L, G, D)
    check(mb.attention_prompt(q, k, v, torch.tensor([0, 1], dtype=torch.int32, device=DEV), cu_k=torch.tensor([0, L], dtype=torch.int32, device=DEV), workspace=workspace), v)
    table, lens = torch.arange(L // page, dtype=torch.int32, device=DEV)[None], torch.tensor([L], dtype=torch.int32, device=DEV)
    pages = [t.view(L // page, page, G, D).transpose(1, 2) for t in (k, v)]
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for said in (1, 1000):
        check(mb.attention_paged(q, *pages, table, lens, cu, said, workspace=workspace), v)
