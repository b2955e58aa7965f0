"""What quant_fp8 makes are two tensors of their own: they can be saved, kept and freed one without the other."""
import io

import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("tile", [1, 128])
@pytest.mark.parametrize("rows,K", [(1, 128), (130, 300), (32, 2048)])
def test_codes_and_scales_can_be_saved(tile, rows, K):
    x = torch.randn(rows, K, device=DEV, generator=torch.Generator(device=DEV).manual_seed(rows))
    q, s = mb.quant_fp8(x, tile=tile)
    file = io.BytesIO()
    torch.save({"q": q, "s": s}, file)
    file.seek(0)
    back = torch.load(file)
    assert torch.equal(back["q"].view(torch.uint8), q.view(torch.uint8)) and torch.equal(back["s"], s)
    assert q.untyped_storage().data_ptr() != s.untyped_storage().data_ptr()
    assert s.untyped_storage().nbytes() == s.numel() * 4  # keeping the scales keeps no codes


def test_one_given_and_one_made():
    x = torch.randn(40, 200, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    q, s = mb.quant_fp8(x)
    q2, s2 = mb.quant_fp8(x, out=torch.empty_strided(q.shape, q.stride(), dtype=q.dtype, device=DEV))  # rows on 16-byte boundaries
    q3, s3 = mb.quant_fp8(x, scales=torch.empty_like(s))
    for a, b in ((q2, s2), (q3, s3)):
        assert torch.equal(a.view(torch.uint8), q.view(torch.uint8)) and torch.equal(b, s)
