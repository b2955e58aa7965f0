"""The feed-forward half of a decoder layer of experts, with a shared expert, in 8-bit floating point.

    python examples/expert_layer.py            # on a B200: a decode step of eight requests, and a prompt

Weights become e4m3 once (quant_fp8 in blocks of 128 x 128).  A step of up to 32 tokens runs its experts as one layer (moe_fp8, or moe4 where they
are packed 4-bit weights); the expert that all tokens share is two products (gemm_fp8) of activations quantized in blocks of 128.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import miori_b200 as mb  # noqa: E402
from miori_b200 import synth  # noqa: E402

EPS = 1e-5
AT_ONCE = 32  # tokens of a layer of experts


def blocked(w):
    """w [rows][K] as (e4m3, scales), stacked where there are several."""
    if w.dim() == 2:
        return mb.quant_fp8(w, tile=128)
    return tuple(torch.stack(t) for t in zip(*(mb.quant_fp8(m, tile=128) for m in w)))


class ExpertLayer:
    """x + experts(norm(x)) + shared(norm(x)), weights of synthetic values; bits: 8, or 4 for the routed experts packed in groups of 64."""

    def __init__(self, hidden, ff, experts, top, shared_ff, device, seed=0, bits=8):
        g = torch.Generator(device=device).manual_seed(seed)
        random = lambda *shape: torch.randn(*shape, generator=g, device=device) * shape[-1] ** -0.5  # noqa: E731
        self.top, self.ff, self.bits = top, ff, bits
        self.norm = (1 + 0.1 * torch.randn(hidden, generator=g, device=device)).to(torch.bfloat16)
        self.router = random(experts, hidden).to(torch.bfloat16)
        self.bias = 0.01 * torch.randn(experts, generator=g, device=device)  # evens out how often an expert is chosen
        if bits == 8:
            self.experts = blocked(random(experts, 2 * ff, hidden)) + blocked(random(experts, hidden, ff))
        else:
            packed = [[synth.make_weight(n, k, 4, 64, seed=seed + 2 * e + i, device=device) for e in range(experts)] for i, (n, k) in enumerate(((2 * ff, hidden), (hidden, ff)))]
            self.experts = tuple(torch.stack(t) for matrices in packed for t in zip(*matrices))
        self.shared = blocked(random(2 * shared_ff, hidden)) + blocked(random(hidden, shared_ff))

    def routed(self, h, workspace):
        """The chosen experts of h bf16 [tokens][hidden], 32 tokens at a time."""
        out = torch.empty(h.shape, device=h.device)
        for i in range(0, h.shape[0], AT_ONCE):
            args = (h[i:i + AT_ONCE], self.router, *self.experts, self.top, workspace)
            options = dict(bias=self.bias, flags=mb.MOE_SIGMOID | mb.MOE_NORM, out=out[i:i + AT_ONCE])
            mb.moe_fp8(*args, **options) if self.bits == 8 else mb.moe4(*args, group=64, **options)
        return out

    def common(self, h):
        """The shared expert of any number of tokens."""
        w_up, s_up, w_down, s_down = self.shared
        gate, up = mb.gemm_fp8(*mb.quant_fp8(h), w_up, s_up).chunk(2, 1)
        return mb.gemm_fp8(*mb.quant_fp8(mb.silu_mul(gate.contiguous(), up.contiguous())), w_down, s_down)

    def __call__(self, x, workspace):
        """x fp32 [tokens][hidden]; returns the residual stream behind the layer."""
        h = mb.rmsnorm(x, self.norm, EPS)
        return x + self.routed(h, workspace) + self.common(h)


def main(device="cuda:0"):
    layer = ExpertLayer(2048, 768, 64, 8, 1536, device)
    workspace = mb.moe_workspace(AT_ONCE, layer.top, layer.ff, device)
    g = torch.Generator(device=device).manual_seed(1)
    prompt = layer(torch.randn(300, 2048, generator=g, device=device), workspace)
    x = torch.randn(8, 2048, generator=g, device=device)
    layer(x, workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # one decode step of all requests
        y = layer(x, workspace)
    begin, end, steps = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True), 50
    begin.record()
    for _ in range(steps):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    assert mb.lib.miori_device_error_poll() == 0 and torch.isfinite(y).all() and torch.isfinite(prompt).all()
    print(f"a layer of 64 experts, 8 for a token, and a shared one: {begin.elapsed_time(end) / steps * 1e3:.1f} us a step of {x.shape[0]} tokens")


if __name__ == "__main__":
    main()
