"""The attention half of a decoder layer over a paged cache, from packed 4-bit weights to the residual.

    python examples/attention_layer.py            # on a B200: three prompts in chunks, then a few decode steps

One step is page_slots (once for all layers), then per layer rmsnorm, the QKV projection, rope_kv, attention_paged, the output
projection and the residual.  Nothing in a step depends on a length on the host, so `decode` is recorded once as a CUDA graph
and replayed while the requests grow.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import miori_b200 as mb  # noqa: E402
from miori_b200 import synth  # noqa: E402

EPS = 1e-5


class PagedCache:
    """Keys and values of one layer after the other, and the page bookkeeping that all layers share."""

    def __init__(self, layers, requests, pages, page, width, kv_heads, dim, device):
        self.k = torch.empty(layers, pages, kv_heads, page, dim, dtype=torch.bfloat16, device=device)
        self.v = torch.empty_like(self.k)
        self.page = page
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.pool = torch.arange(pages, dtype=torch.int32, device=device)
        self.taken = torch.zeros(1, dtype=torch.int32, device=device)
        self.held = torch.zeros(requests, dtype=torch.int32, device=device)

    def step(self, new, tokens):
        """Slots, positions, cu and lengths of a step that adds new[r] tokens to request r, `tokens` rows in all."""
        slots, positions, cu, held, taken = mb.page_slots(self.held, new, self.table, self.pool, self.taken, self.page, tokens)
        self.held.copy_(held)
        self.taken.copy_(taken)
        return slots, positions, cu, held


class AttentionLayer:
    """x + W_o attention(rope(norm_head(W_qkv norm(x)))) with 4-bit weights of synthetic values."""

    def __init__(self, hidden, heads, kv_heads, dim, device, seed=0, theta=1e6, group=64):
        self.heads, self.kv_heads, self.dim, self.group = heads, kv_heads, dim, group
        self.qkv = synth.make_weight((heads + 2 * kv_heads) * dim, hidden, 4, group, seed=seed, device=device)
        self.o = synth.make_weight(hidden, heads * dim, 4, group, seed=seed + 1, device=device)
        self.caches = [mb.dequant4_cache(*w, group=group) for w in (self.qkv, self.o)]
        g = torch.Generator().manual_seed(seed)
        self.norm, self.norm_q, self.norm_k = ((1 + 0.1 * torch.randn(n, generator=g)).to(device, torch.bfloat16) for n in (hidden, dim, dim))
        self.turns, self.axes = mb.rope_turns(dim, theta=theta, device=device)

    def project(self, i, h):
        """Rows of a decode step through linear4, of a prompt through the GEMM on the bf16 cache."""
        w = (self.qkv, self.o)[i]
        if h.shape[0] <= 32:
            return mb.linear4(*w, self.caches[i], h, group=self.group)
        return mb.gemm_bf16_cache(h, self.caches[i], w[0].shape[0])

    def __call__(self, x, k_cache, v_cache, table, slots, positions, cu, lens, max_new, workspace):
        """x fp32 [tokens][hidden]; returns the residual stream behind the layer."""
        h = mb.rmsnorm(x, self.norm, EPS)
        qkv = self.project(0, h)
        q = mb.rope_kv(qkv, self.turns, positions, slots, k_cache, v_cache, self.heads, axes=self.axes, gamma_q=self.norm_q, gamma_k=self.norm_k, eps=EPS)
        a = mb.attention_paged(q, k_cache, v_cache, table, lens, cu, max_new, workspace=workspace)
        return x + self.project(1, a.view(x.shape[0], -1))


def run_step(layers, cache, x, new, max_new, workspace):
    """All layers over the tokens of one step."""
    slots, positions, cu, lens = cache.step(new, x.shape[0])
    for i, layer in enumerate(layers):
        x = layer(x, cache.k[i], cache.v[i], cache.table, slots, positions, cu, lens, max_new, workspace)
    return x


def main(device="cuda:0"):
    layers = [AttentionLayer(2048, 16, 4, 128, device, seed=10 * i) for i in range(4)]
    prompts, chunk, steps = [700, 33, 1500], 512, 16
    cache = PagedCache(len(layers), len(prompts), pages=200, page=16, width=128, kv_heads=4, dim=128, device=device)
    workspace = mb.attention_workspace(device)
    g = torch.Generator(device=device).manual_seed(1)
    left = list(prompts)
    while any(left):  # prompts, a chunk of each at a time
        new = [min(chunk, n) for n in left]
        left = [n - m for n, m in zip(left, new)]
        run_step(layers, cache, torch.randn(sum(new), 2048, generator=g, device=device), torch.tensor(new, dtype=torch.int32, device=device), max(new), workspace)
    x, one = torch.randn(len(prompts), 2048, generator=g, device=device), torch.ones(len(prompts), dtype=torch.int32, device=device)
    run_step(layers, cache, x, one, 1, workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # one decode step of all requests
        y = run_step(layers, cache, x, one, 1, workspace)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(steps):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    # a recorded step cannot stop where the pool runs out: positions without a page are then seen by no token, and `taken` says so
    assert int(cache.taken) <= cache.pool.numel(), "not enough pages"
    assert mb.lib.miori_device_error_poll() == 0 and torch.isfinite(y).all()
    print(f"{len(layers)} attention layers, positions {cache.held.tolist()}: {begin.elapsed_time(end) / steps * 1e3:.1f} us a decode step, "
          f"{int(cache.taken)} pages of {cache.page} taken")


if __name__ == "__main__":
    main()
