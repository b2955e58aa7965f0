"""Layers of experts with as many lists of tokens as 32 tokens of 16 of 256 experts can make, over rows of several units.

A warp of the second product keeps a cell for every list that it meets, so these are the calls that ask most of its shared memory; and what it keeps is laid down
from a formula, which is looked through here for every number of units."""
import os
import re

import pytest
import torch

import miori_b200 as mb
import test_moe_gpu as moe
from conftest import ROOT

DEV = "cuda:0"


def most_met(entries, units, workers=64):
    """The most entries that one of the warps meets when their units are dealt to them evenly, by counting."""
    total = entries * units
    return max((total * (w + 1) // workers - 1) // units - total * w // workers // units + 1 for w in range(workers) if total * w // workers < total * (w + 1) // workers)


def test_the_formula_covers_every_deal():
    """And reserves, for some, more cells than if every entry were one unit: the room that is asked for at compile time is that of all of them."""
    code = open(os.path.join(ROOT, "miori_b200", "csrc", "moe.cuh")).read()
    assert re.search(r"segments_of\(uint32_t all_units, uint32_t units\)", code)

    def segments(entries, units):
        return (max(-(-entries * units // 64), 1) + units - 2) // units + 1

    for entries in [*range(1, 330, 7), 288, 320]:
        for units in [*range(1, 40), 255, 256, 512]:
            assert most_met(entries, units) <= segments(entries, units), (entries, units)
    assert segments(288, 3) == 6 > -(-320 // 64)
    host = open(os.path.join(ROOT, "miori_b200", "csrc", "moe.cu")).read()
    assert "static_assert(SMEM - Stage<FMT>::ring(Stage<FMT>::DOWN) >= ONE_TILE<FMT>" in host and re.search(r"segments_of\(MAX_\w*ENTRIES \* units, units\)", host)


def crowded(bits, group, popular, tokens_each, H, F, seed):
    """32 tokens of 16 experts each: `popular` of the 256 have tokens_each tokens, all others one."""
    x, router, ws, _ = moe.make(bits, group, 32, 256, H, F, seed)
    of_popular = popular * tokens_each // 32
    picks = [[(t * (popular // 32) + j) % popular for j in range(of_popular)] + [popular + t * (16 - of_popular) + j for j in range(16 - of_popular)] for t in range(32)]
    counts = torch.bincount(torch.tensor(picks).flatten(), minlength=256)
    assert counts[:popular].eq(tokens_each).all() and counts[popular:].eq(1).all()
    x[:, :32] = torch.eye(32, device=DEV) * 4
    router[:] = 0
    for t, row in enumerate(picks):
        router[row, t] = (0.5 + 0.1 * torch.arange(16, device=DEV)).to(torch.bfloat16)
    return x, router, ws, picks


@pytest.mark.gpu
@pytest.mark.parametrize("popular,tokens_each", [(32, 9), (64, 5)])
@pytest.mark.parametrize("bits,group,F", [(4, 32, 768), (4, 32, 1024), (4, 64, 512), (4, 64, 1280), (8, 128, 384), (8, 128, 640)])
def test_the_most_lists_over_several_units(bits, group, F, popular, tokens_each):
    x, router, ws, picks = crowded(bits, group, popular, tokens_each, 128, F, popular + F)
    lists = moe.choice(x, router, 16, None, True, False, 1.0)
    assert all(sorted(e for e, _ in row) == sorted(p) for row, p in zip(lists, picks))
    moe.check(x, router, ws, bits, group, 16, None, mb.MOE_SIGMOID)
    moe.check(x, router, ws, bits, group, 16, None, mb.MOE_SIGMOID | mb.MOE_NORM | mb.OUT_BF16)
