"""The attention operators together, as a layer uses them: prompts in chunks over the page cache, then decode steps, against the
same layer in plain fp32 over contiguous keys, and against packed prompts without a cache."""
import importlib.util
import math
import os

import pytest
import torch

import miori_b200 as mb
from conftest import ROOT, assert_close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def example():
    spec = importlib.util.spec_from_file_location("attention_layer", os.path.join(ROOT, "examples", "attention_layer.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def dense(w, group):
    return mb.dequant4_rowmajor(*w, group=group).float()


class Plain:
    """The same layer in fp32; keys and values as the cache holds them."""

    def __init__(self, layer):
        self.l, self.qkv, self.o = layer, dense(layer.qkv, layer.group), dense(layer.o, layer.group)
        half = layer.dim // 2
        self.freq = torch.tensor([1e6 ** (-j / half) for j in range(half)], dtype=torch.float64, device=DEV)
        self.k, self.v = [], []

    def __call__(self, x):
        l, n, first = self.l, x.shape[0], sum(t.shape[0] for t in self.k)
        norm = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-5) * w.float()  # noqa: E731
        y = (norm(x, l.norm).bfloat16().float() @ self.qkv.T).view(n, -1, l.dim)
        q, k, v = y.split([l.heads, l.kv_heads, l.kv_heads], 1)
        angle = (torch.arange(first, first + n, device=DEV).double()[:, None] * self.freq)[:, None]
        cos, sin = angle.cos().float(), angle.sin().float()

        def turned(t, w):
            a, b = norm(t, w).chunk(2, -1)
            return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).bfloat16().float()

        self.k.append(turned(k, l.norm_k)), self.v.append(v.bfloat16().float())
        kk, vv = (torch.cat(t).repeat_interleave(l.heads // l.kv_heads, 1) for t in (self.k, self.v))
        s = torch.einsum("nhd,lhd->hnl", turned(q, l.norm_q), kk) / math.sqrt(l.dim)
        hidden = torch.arange(kk.shape[0], device=DEV)[None] > torch.arange(first, first + n, device=DEV)[:, None]
        a = torch.einsum("hnl,lhd->nhd", torch.softmax(s.masked_fill(hidden, -math.inf), -1), vv).reshape(n, -1)
        return x + a.bfloat16().float() @ self.o.T


def test_chunks_and_steps():
    ex = example()
    layers = [ex.AttentionLayer(512, 8, 2, 64, DEV, seed=s) for s in (0, 10)]
    cache = ex.PagedCache(2, 3, pages=64, page=16, width=24, kv_heads=2, dim=64, device=DEV)
    cache.k.fill_(math.nan), cache.v.fill_(math.inf)  # what nobody has written has no influence
    ws = mb.attention_workspace(DEV)
    plain = [[Plain(l) for l in layers] for _ in range(3)]
    g = torch.Generator(device=DEV).manual_seed(3)
    steps = ([100, 7, 0], [60, 0, 90], [1, 1, 1], [1, 1, 1], [4, 1, 2], [1, 0, 130])
    for new in steps:
        x = torch.randn(sum(new), 512, generator=g, device=DEV)
        y = ex.run_step(layers, cache, x, torch.tensor(new, dtype=torch.int32, device=DEV), max(new), ws)
        at = 0
        for r, n in enumerate(new):
            if n:
                want = x[at:at + n]
                for p in plain[r]:
                    want = p(want)
                assert_close(y[at:at + n].cpu().numpy(), want.cpu().numpy(), what=f"step {new}, request {r}")
            at += n
    held = [sum(new[r] for new in steps) for r in range(3)]
    assert cache.held.tolist() == held and int(cache.taken) == sum(-(-n // 16) for n in held)
    assert mb.lib.miori_device_error_poll() == 0


def test_a_prompt_over_the_cache_and_packed_agree():
    """The same heads through attention_paged in one chunk and through attention_prompt: within a rounding of each other."""
    g = torch.Generator(device=DEV).manual_seed(4)
    lengths, H, G, D, page = [300, 1, 270], 8, 2, 128, 32
    T = sum(lengths)
    cu = torch.tensor([0] + lengths, device=DEV).cumsum(0).to(torch.int32)
    new = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    table = torch.full((3, 12), -1, dtype=torch.int32, device=DEV)
    slots, positions, cu2, lens, _ = mb.page_slots(torch.zeros_like(new), new, table, torch.arange(24, dtype=torch.int32, device=DEV).flip(0).contiguous(),
                                                   torch.zeros(1, dtype=torch.int32, device=DEV), page, T)
    assert torch.equal(cu, cu2)
    qkv = torch.randn(T, (H + 2 * G) * D, generator=g, device=DEV)
    turns, axes = mb.rope_turns(D, theta=1e4, device=DEV)
    pages = torch.empty(2, 24, G, page, D, dtype=torch.bfloat16, device=DEV)
    q = mb.rope_kv(qkv, turns, positions, slots, pages[0], pages[1], H, axes=axes)
    # a cache of pages of one position, a page a token, is the packed tensor
    packed = torch.empty(2, T, G, D, dtype=torch.bfloat16, device=DEV)
    view = packed.view(2, T, G, 1, D)
    q2 = mb.rope_kv(qkv, turns, positions, torch.arange(T, dtype=torch.int32, device=DEV), view[0], view[1], H, axes=axes)
    assert torch.equal(q, q2)
    ws = mb.attention_workspace(DEV)
    a = mb.attention_paged(q, pages[0], pages[1], table, lens, cu, max(lengths), workspace=ws).float()
    b = mb.attention_prompt(q, packed[0], packed[1], cu, workspace=ws).float()
    # both are within 2^-8 (|o| + sum w |v|) of the formula's value; |v| is below 6 here
    assert ((a - b).abs() <= 2 * 2.0 ** -8 * (b.abs() + 6.0)).all()
    assert_close(a.cpu().numpy(), b.cpu().numpy())


def test_the_example_runs(capsys):
    example().main(DEV)
    assert "us a decode step" in capsys.readouterr().out
