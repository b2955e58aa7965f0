"""What holds for one kernel of gemm_fp8 by size is looked at for every one of them, chosen by the tuning bits: what spoils an element spoils no other, and rows may lie further
apart than 32 bits count, in bytes and in elements."""
import pytest
import torch

import miori_b200 as mb
import test_fp8_gpu as fp8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# few rows in tiles of 16, 32, 64, 128, whole and with K in halves; pairs of 128 and of 256 columns
KERNELS = [kind << 20 | halves << 23 for kind in (1, 2, 3, 4) for halves in (0, 1)] + [5 << 20, 6 << 20]


@pytest.mark.parametrize("tune", KERNELS, ids=hex)
@pytest.mark.parametrize("M,N", [(20, 130), (300, 400), (257, 513)])
@pytest.mark.parametrize("flags", [0, 1])
def test_a_nan_or_an_infinite_scale_stays_in_its_row_and_column(tune, M, N, flags):
    a, sa, w, sw = fp8.operands(M, N, 256, 6)
    a.view(torch.uint8)[7, 130] = 0x7F
    w.view(torch.uint8)[N - 2, 3] = 0x7F
    sa[9, 1] = float("inf")
    last = M - 1
    sa[last, 0] = float("nan")
    got = mb.gemm_fp8(a, sa, w, sw, flags=tune | flags)
    want = torch.zeros((M, N), dtype=torch.bool, device=DEV)
    want[[7, 9, last]], want[:, N - 2] = True, True
    assert torch.equal(~torch.isfinite(got), want)
    clean = fp8.operands(M, N, 256, 6)
    rows, cols = [m for m in range(M) if m not in (7, 9, last)], [n for n in range(N) if n != N - 2]
    assert torch.equal(got[rows][:, cols], mb.gemm_fp8(*clean, flags=tune | flags)[rows][:, cols])
    # a block of w whose scale is none: its 128 columns, in the last block those up to N
    a, sa, w, sw = clean
    sw[-1, 1] = float("inf")
    got = mb.gemm_fp8(a, sa, w, sw, flags=tune | flags)
    want = torch.zeros((M, N), dtype=torch.bool, device=DEV)
    want[:, (N - 1) // 128 * 128:] = True
    assert torch.equal(~torch.isfinite(got), want)
    assert mb.lib.miori_device_error_poll() == 0


def far(rows, cols, dtype, beyond=2 ** 32):
    """[rows][cols] whose last row begins `beyond` elements behind the first, or more; rows on 16-byte boundaries."""
    pitch = (beyond // (rows - 1) // 16 + 1) * 16
    whole = torch.empty((rows - 1) * pitch + cols + 16, dtype=dtype, device=DEV)
    t = whole.as_strided((rows, cols), (pitch, 1))
    assert t.stride(0) * (rows - 1) >= 2 ** 32 and pitch < 2 ** 40
    return t


@pytest.mark.parametrize("tune", KERNELS, ids=hex)
@pytest.mark.parametrize("N,flags", [(200, 1), (203, 1), (200, 0), (201, 0)])  # rows of C that a copy by TMA can describe, and others
def test_rows_of_c_beyond_32_bits(tune, N, flags):
    M = 300
    ops = fp8.operands(M, N, 256, 11)
    out = far(M, N + 8, torch.bfloat16 if flags else torch.float32)
    out.fill_(2.0)
    got = mb.gemm_fp8(*ops, flags=tune | flags, out=out[:, :N])
    fp8.close(got, *ops)
    assert torch.equal(got, mb.gemm_fp8(*ops, flags=tune | flags))
    assert bool((out[:, N:] == 2).all())
    assert mb.lib.miori_device_error_poll() == 0


@pytest.mark.parametrize("tune", KERNELS, ids=hex)
def test_operands_and_scales_beyond_32_bits(tune):
    M, N, K = 290, 260, 300
    a, sa, w, sw = ops = fp8.operands(M, N, K, 12)
    want = mb.gemm_fp8(*ops, flags=tune)
    fp8.close(want, *ops)
    far_a, far_w = (far(t.shape[0], K, torch.uint8).view(torch.float8_e4m3fn) for t in (a, w))
    far_a.view(torch.uint8).copy_(fp8.bits(a)), far_w.view(torch.uint8).copy_(fp8.bits(w))
    assert torch.equal(mb.gemm_fp8(far_a, sa, far_w, sw, flags=tune), want)
    del far_a, far_w
    far_sa, far_sw = (far(t.shape[0], t.shape[1], torch.float32) for t in (sa, sw))
    far_sa.copy_(sa), far_sw.copy_(sw)
    assert torch.equal(mb.gemm_fp8(a, far_sa, w, far_sw, flags=tune), want)
    assert mb.lib.miori_device_error_poll() == 0


@pytest.mark.parametrize("tile", [1, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quant_beyond_32_bits(tile, dtype):
    """Rows of x, of the codes and of the scales."""
    rows, K = 260, 300
    x = torch.randn(rows, K, device=DEV, generator=torch.Generator(device=DEV).manual_seed(13)).to(dtype)
    want = mb.quant_fp8(x, tile=tile)
    fp8.same(want, fp8.oracle_quant(x, tile))
    far_x = far(rows, K, dtype)
    far_x.copy_(x)
    fp8.same(mb.quant_fp8(far_x, tile=tile), want)
    del far_x
    q, s = far(rows, K, torch.uint8).view(torch.float8_e4m3fn), far(want[1].shape[0], want[1].shape[1], torch.float32)
    fp8.same(mb.quant_fp8(x, tile=tile, out=q, scales=s), want)
