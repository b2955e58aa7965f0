"""The operators in 8-bit floating point and the layers of experts together, as a decoder layer uses them, against the same layer in 64 bits.

The routed experts take activations without quantizing them: within 2^-9 as a whole (2^-11 of the activation between the products, weights of the same values on
both sides).  The shared expert's are rounded to e4m3 twice: each factor's rounding is off by up to 2^-4, 2^-4 / sqrt(3) = 0.036 in the mean, and the weights are the same on
both sides; the first product's error, 0.036, goes through silu(g) u, whose relative slopes add up to at most 1.5 and 1: 0.065; with the second rounding 0.075.  Twice that is allowed."""
import importlib.util
import os

import pytest
import torch

import miori_b200 as mb
from conftest import ROOT

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def example():
    spec = importlib.util.spec_from_file_location("expert_layer", os.path.join(ROOT, "examples", "expert_layer.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def unblocked(w, s):
    return w.double() * s.double().repeat_interleave(128, -2)[..., :w.shape[-2], :].repeat_interleave(128, -1)[..., :w.shape[-1]]


class Plain:
    """The layer in 64 bits."""

    def __init__(self, layer):
        self.l = layer
        if layer.bits == 8:
            self.up, self.down = unblocked(*layer.experts[:2]), unblocked(*layer.experts[2:])
        else:
            self.up, self.down = (torch.stack([mb.dequant4_rowmajor(*(t[e] for t in w), group=64) for e in range(w[0].shape[0])]).double()
                                  for w in (layer.experts[:3], layer.experts[3:]))
        self.shared = unblocked(*layer.shared[:2]), unblocked(*layer.shared[2:])

    @staticmethod
    def ff(x, up, down):
        g, u = (up @ x).chunk(2)
        return down @ (torch.nn.functional.silu(g) * u)

    def parts(self, h):
        h = h.double()
        p = torch.sigmoid(h @ self.l.router.double().T)
        chosen = torch.topk(p + self.l.bias.double(), self.l.top).indices
        weights = p.gather(1, chosen)
        weights = weights / weights.sum(1, keepdim=True)
        routed = torch.stack([sum(w * self.ff(x, self.up[e], self.down[e]) for e, w in zip(c.tolist(), ws)) for x, c, ws in zip(h, chosen, weights)])
        if self.l.bits == 4:  # as dequant4_rowmajor has them, rounded to bf16: within 2^-8 of the operator's
            return routed, 2.0 ** -7, torch.stack([self.ff(x, *self.shared) for x in h])
        return routed, 2.0 ** -9, torch.stack([self.ff(x, *self.shared) for x in h])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("tokens", [1, 6, 32, 70])
def test_layer(bits, tokens):
    ex = example()
    layer = ex.ExpertLayer(512, 256, 16, 4, 384, DEV, seed=tokens, bits=bits)
    plain, workspace = Plain(layer), mb.moe_workspace(32, 4, 256, DEV)
    x = torch.randn(tokens, 512, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    h = mb.rmsnorm(x, layer.norm, ex.EPS)
    routed, room, shared = plain.parts(h)
    off = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert off(layer.routed(h, workspace), routed) < room
    assert off(layer.common(h), shared) < 0.15
    y = layer(x, workspace)
    assert torch.equal(y, x + layer.routed(h, workspace) + layer.common(h))
    # recorded, and replayed for other tokens
    given = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = layer(given, workspace)
    graph.replay()
    assert torch.equal(z, y)
    given.copy_(-x.flip(0))
    graph.replay()
    assert torch.equal(z, layer(-x.flip(0), workspace))
    assert mb.lib.miori_device_error_poll() == 0


def test_the_example_runs(capsys):
    example().main(DEV)
    assert "us a step of 8 tokens" in capsys.readouterr().out
