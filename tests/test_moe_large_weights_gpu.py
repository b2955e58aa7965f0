"""Experts whose weights begin beyond 2^32 bytes, in both formats and both products."""
import pytest
import torch

import miori_b200 as mb
import test_moe_gpu as moe

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("bits,group,E,H,F", [(4, 64, 224, 7168, 5632), (4, 32, 224, 7168, 5632), (8, 128, 112, 7168, 5616)])
def test_experts_beyond_32_bits(bits, group, E, H, F):
    chosen = [0, E // 2, E - 1]
    x, router, few, _ = moe.make(bits, group, 3, len(chosen), H, F, E, bias=False)
    ws = [torch.empty((E, *t.shape[1:]), dtype=t.dtype, device=DEV) for t in few]  # of nobody's experts: whatever lies there
    for w, t in zip(ws, few):
        w[chosen] = t
    for w in (ws[0], ws[len(ws) // 2]):
        assert (E - 1) * w[0].numel() * w.element_size() > 2 ** 32
    wide = torch.zeros((E, H), dtype=torch.bfloat16, device=DEV)
    wide[chosen] = router
    bias = torch.full((E,), -float("inf"), device=DEV)
    bias[chosen] = 0
    flags = mb.MOE_SIGMOID | mb.MOE_NORM
    got = moe.run(x, wide, ws, bits, group, 2, bias, flags)
    # not the bits of a layer of these three alone: a router of so many experts adds up K in other parts
    want, tol = moe.oracle(x, router, few, bits, group, 2, torch.zeros(3, device=DEV), True, True, 1.0)
    assert bool(((got.double() - want).abs() <= tol).all())
    assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -11
    assert mb.lib.miori_device_error_poll() == 0
