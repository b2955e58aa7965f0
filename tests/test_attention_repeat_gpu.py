"""The same call again and again, alone and beside another on a stream of its own: always the same bits, whatever else the GPU does."""
import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV).to(torch.bfloat16)


def prompt_call(seed, lengths, H, G, D):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = sum(lengths)
    q, k, v, ws = rand(g, T, H, D), rand(g, T, G, D), rand(g, T, G, D), mb.attention_workspace(DEV)
    cu = torch.tensor([0] + lengths, device=DEV).cumsum(0).to(torch.int32)
    return lambda: mb.attention_prompt(q, k, v, cu, workspace=ws)


def paged_call(seed, held, new, H, G, D, page=16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    R, width = len(held), -(-(max(held) + new) // page)
    cache, q, ws = rand(g, 2, R * width, G, page, D), rand(g, R * new, H, D), mb.attention_workspace(DEV)
    table = torch.randperm(R * width, generator=g, device=DEV).to(torch.int32).view(R, width)
    lens, cu = torch.tensor([h + new for h in held], dtype=torch.int32, device=DEV), torch.arange(0, (R + 1) * new, new, dtype=torch.int32, device=DEV)
    return lambda: mb.attention_paged(q, cache[0], cache[1], table, lens, cu, new, workspace=ws)


CALLS = {
    "prompts 128": lambda: prompt_call(1, [3000, 20, 1111, 129, 64], 8, 2, 128),
    "prompts 64": lambda: prompt_call(2, [3000, 20, 1111, 129, 64], 16, 4, 64),
    "one row tile an item": lambda: prompt_call(3, [2000] + [33] * 20 + [500], 4, 1, 128),  # some items have a second row tile, others none
    "short prompts": lambda: prompt_call(4, [77, 130, 1, 60], 16, 4, 128),
    "chunks 128": lambda: paged_call(5, [2000, 0, 900], 100, 8, 2, 128),
    "chunks 64": lambda: paged_call(6, [2000, 0, 900], 100, 8, 2, 64),
    "decode 128": lambda: paged_call(7, [20000, 5, 900], 1, 16, 4, 128),
    "drafts 64": lambda: paged_call(8, [9000, 5, 900], 5, 32, 8, 64),
}


@pytest.mark.parametrize("name", CALLS)
def test_again_and_again(name):
    call = CALLS[name]()
    want = call()
    outs = [call() for _ in range(30)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert mb.lib.miori_device_error_poll() == 0


@pytest.mark.parametrize("pair", [("prompts 128", "decode 128"), ("prompts 64", "chunks 128"), ("drafts 64", "decode 128"), ("short prompts", "chunks 64"),
                                  ("prompts 128", "prompts 64"), ("decode 128", "decode 128")])
def test_two_streams_with_workspaces_of_their_own(pair):
    calls = [CALLS[name]() for name in pair]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(calls[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    assert mb.lib.miori_device_error_poll() == 0
