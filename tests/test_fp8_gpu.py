"""quant_fp8 bit for bit against its definition, gemm_fp8 against 64-bit sums.

A product's tolerance, element by element.  S = sum_b sa sw sum |a w| bounds every partial sum.  A product of two e4m3 is exact; an MMA adds 32 of
them and the running sum, each cut off no earlier than at 2^-24 of the largest: 33 * 2^-24 of S at most, four MMAs a block.  The scale (one rounding), the
product with it and the sum over blocks: (blocks + 3) * 2^-24 of S.  bf16 outputs: 2^-8 of the value on top."""
import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP8 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // 128)


def oracle_quant(x, tile):
    """The definition, one operation after the other in fp32; NaN does not count for the largest."""
    rows, K = x.shape
    R = -(-rows // tile)
    v = torch.nn.functional.pad(x.float(), (0, blocks(K) * 128 - K, 0, R * tile - rows)).view(R, tile, blocks(K), 128)
    top = v.nan_to_num(nan=0.0, posinf=float("inf"), neginf=float("-inf")).abs().amax((1, 3)).clamp(min=2.0 ** -100)
    most = torch.full_like(top, 448.0)  # a plain number would be divided by as a product with its reciprocal
    q = (v * (most / top)[:, None, :, None]).to(FP8).flatten(2).flatten(0, 1)
    return q[:rows, :K], top / most


def bits(q):
    return q.contiguous().view(torch.uint8)


def same(got, want):
    for g, w in ((bits(got[0]), bits(want[0])), (got[1], want[1])):
        # every NaN is the same to us
        nan = torch.isnan(got[0].float()) & torch.isnan(want[0].float()) if g.dtype == torch.uint8 else torch.zeros_like(g, dtype=torch.bool)
        assert bool(((g == w) | nan).all()), (g.shape, int((g != w).sum()))


@pytest.mark.parametrize("tile", [1, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 128), (3, 130), (32, 2048), (127, 127), (129, 1440), (257, 264), (300, 4097), (1000, 2048)])
def test_quant(rows, K, dtype, tile):
    g = torch.Generator(device=DEV).manual_seed(rows * 7 + K)
    x = (torch.randn(rows, K, generator=g, device=DEV) * torch.exp(4 * torch.randn(rows, 1, generator=g, device=DEV))).to(dtype)
    same(mb.quant_fp8(x, tile=tile), oracle_quant(x, tile))


@pytest.mark.parametrize("tile", [1, 128])
def test_quant_of_unusual_values(tile):
    x = torch.randn(260, 500, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    x[0] = 0.0
    x[1] *= 1e-42          # subnormal
    x[2, :128] = 448.0
    x[2, 128:256] = 464.0  # as 448 does, it has to come out as 448 times its scale
    x[3] *= 1e38
    x[4, 3] = float("nan")
    x[5, 200] = float("inf")
    x[130, 7] = float("-inf")
    x[131:] = 0.0
    for v in (x, x.to(torch.bfloat16)):
        q, s = mb.quant_fp8(v, tile=tile)
        same((q, s), oracle_quant(v, tile))
    q, s = mb.quant_fp8(torch.zeros(5, 70, device=DEV), tile=tile)
    assert not bits(q).any() and bool((s > 0).all())


@pytest.mark.parametrize("tile", [1, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quant_of_views_into_views(tile, dtype):
    """Rows of x that begin nowhere in particular, rows of q in a wider tensor, scales with columns outermost; the rest stays."""
    g = torch.Generator(device=DEV).manual_seed(3)
    whole = torch.randn(140, 333, generator=g, device=DEV).to(dtype)
    for x in (whole[:, 3:300], whole[1:139:2, :257], whole[5:6]):
        rows, K = x.shape
        out = torch.full((rows, 512), 1.5, device=DEV).to(FP8)
        scales = torch.full((blocks(K) + 1, -(-rows // tile) + 2), -7.0, device=DEV)
        q, s = mb.quant_fp8(x, tile=tile, out=out[:, 16:16 + K], scales=scales[:blocks(K), :-(-rows // tile)].T)
        same((q, s), oracle_quant(x, tile))
        assert q.data_ptr() == out.data_ptr() + 16
        assert bool((out[:, :16].float() == 1.5).all()) and bool((out[:, 16 + K:].float() == 1.5).all())
        assert bool((scales[-1] == -7).all()) and bool((scales[:, -2:] == -7).all())


def operands(M, N, K, seed, spread=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=DEV)
    if spread:
        x = x * torch.exp(torch.randn(M, 1, generator=g, device=DEV)) * torch.exp(torch.randn(1, K, generator=g, device=DEV))
    a, sa = oracle_quant(x, 1)
    w, sw = oracle_quant(torch.randn(N, K, generator=g, device=DEV) * torch.exp(torch.randn(N, 1, generator=g, device=DEV)), 128)

    def pitched(q):  # rows on 16-byte boundaries
        wide = torch.zeros(q.shape[0], (K + 15) // 16 * 16, dtype=torch.uint8, device=DEV).view(FP8)
        wide.view(torch.uint8)[:, :K] = bits(q)
        return wide[:, :K]
    return pitched(a), sa, pitched(w), sw


def exact(a, sa, w, sw):
    """(C, S) in 64 bits."""
    C = torch.zeros(a.shape[0], w.shape[0], dtype=torch.float64, device=DEV)
    S = torch.zeros_like(C)
    of = torch.arange(w.shape[0], device=DEV) // 128
    for b in range(blocks(a.shape[1])):
        x, y = (t[:, b * 128:(b + 1) * 128].double() for t in (a, w))
        scale = sa[:, b].double()[:, None] * sw[of, b].double()
        C += scale * (x @ y.T)
        S += scale.abs() * (x.abs() @ y.abs().T)
    return C, S


def close(got, a, sa, w, sw):
    C, S = exact(a, sa, w, sw)
    tol = S * ((4 * 33 + blocks(a.shape[1]) + 3) * 2.0 ** -24)
    if got.dtype == torch.bfloat16:
        tol = tol + C.abs() * 2.0 ** -8
    bad = (got.double() - C).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())
    if got.dtype == torch.float32:
        assert float((got.double() - C).norm() / C.norm()) < 2e-5


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 2048, 2048), (1, 16384, 2048), (2, 130, 100), (5, 2048, 8192), (8, 5003, 1440), (16, 128, 128), (17, 256, 129), (31, 4096, 2000),
                                   (33, 1000, 640), (64, 2048, 2048), (77, 5003, 1440), (100, 2048, 8192), (128, 16384, 2048), (129, 300, 400), (200, 2048, 2048),
                                   (255, 4096, 1440), (257, 16384, 256), (300, 16384, 128), (1024, 2048, 8192), (1000, 9999, 272), (2000, 5000, 130), (4096, 4096, 512)])
@pytest.mark.parametrize("flags", [0, 1])
def test_gemm(M, N, K, flags):
    ops = operands(M, N, K, M + N + K)
    close(mb.gemm_fp8(*ops, flags=flags), *ops)


@pytest.mark.parametrize("M,N", [(3, 100), (40, 333), (150, 700), (2500, 2100)])
@pytest.mark.parametrize("flags", [0, 1])
def test_gemm_of_views_into_views(M, N, flags):
    """Operands, scales and output inside wider tensors, the output's rows on any boundary; the rest of it stays."""
    K = 300
    a, sa, w, sw = operands(M, N, K, 5)
    wide_a, wide_w = torch.full((M, 512), 0x7F, dtype=torch.uint8, device=DEV), torch.full((N, 368), 0x7F, dtype=torch.uint8, device=DEV)  # NaN all around
    wide_a[:, 32:32 + K], wide_w[:, 16:16 + K] = bits(a), bits(w)
    sat = sa.T.contiguous().T
    swt = torch.full((sw.shape[0], 7), float("nan"), device=DEV)
    swt[:, 1:7:2] = sw
    dt = torch.bfloat16 if flags else torch.float32
    out = torch.full((M, N + 21), 3.0, dtype=dt, device=DEV)
    for first in (0, 3):
        got = mb.gemm_fp8(wide_a.view(FP8)[:, 32:32 + K], sat, wide_w.view(FP8)[:, 16:16 + K], swt[:, 1:7:2], flags=flags, out=out[:, first:first + N])
        close(got, a, sa, w, sw)
        assert bool((out[:, :first] == 3).all()) and bool((out[:, first + N:] == 3).all())
        out.fill_(3.0)


def test_gemm_spreads_no_nan():
    """A NaN, or an infinite scale, stays in its row and its column."""
    a, sa, w, sw = operands(300, 400, 256, 6)
    a.view(torch.uint8)[7, 130] = 0x7F
    w.view(torch.uint8)[200, 3] = 0x7F
    sa[9, 1] = float("inf")
    for M in (20, 300):
        got = mb.gemm_fp8(a[:M], sa[:M], w, sw)
        bad = ~torch.isfinite(got)
        want = torch.zeros_like(bad)
        want[7], want[:, 200], want[9] = True, True, True
        assert bool((bad == want).all())


def test_gemm_repeats_and_rows_agree():
    """The same bits every time, in a graph and on another stream."""
    for M, N, K in ((3, 2048, 2048), (70, 2048, 1440), (1500, 4096, 512)):
        ops = operands(M, N, K, 8)
        first = mb.gemm_fp8(*ops)
        assert all(torch.equal(first, mb.gemm_fp8(*ops)) for _ in range(3))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = mb.gemm_fp8(*ops)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(first, other)
        out = torch.zeros_like(first)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q = mb.gemm_fp8(*ops, out=out)
        out.zero_()
        graph.replay()
        assert torch.equal(first, q)


def test_a_projection_in_blocks():
    """From packed weights to a product as a program runs it, with launches that may overlap: the error is what three mantissa bits cost."""
    from miori_b200 import synth
    q, s, b = synth.make_weight(1024, 2048, 4, 64, seed=3, device=DEV)
    dense = mb.dequant4_rowmajor(q, s, b, group=64)
    w, sw = mb.quant_fp8(dense, tile=128)
    gamma = torch.ones(2048, dtype=torch.bfloat16, device=DEV)
    for M in (1, 40, 500):
        x = torch.randn(M, 2048, device=DEV, generator=torch.Generator(device=DEV).manual_seed(M))
        n = mb.rmsnorm(x, gamma, 1e-5, mb.LAUNCH_PDL)
        a, sa = mb.quant_fp8(n)
        C = mb.gemm_fp8(a, sa, w, sw)
        close(C, a, sa, w, sw)
        want = n.double() @ dense.double().T
        # each factor off by 2^-4 of itself at most, 2^-4 / sqrt(3) on average over a binade, of either sign
        assert float((C.double() - want).norm() / want.norm()) < 2 ** 0.5 * 2.0 ** -4
    assert mb.lib.miori_device_error_poll() == 0


FEW, PAIRS = [(mp, cs) for mp in (1, 2, 3, 4) for cs in (0, 1, 2, 3)], [(5, 0), (6, 0)]  # as the tuning bits have them


@pytest.mark.parametrize("kind,log_slices", FEW + PAIRS)
def test_every_kernel_takes_every_size(kind, log_slices):
    """Each tile and split, chosen by the tuning bits rather than by size: the same products within the same tolerance."""
    tune = kind << 20 | log_slices << 23
    for M, N, K in ((1, 1, 16), (9, 130, 1100), (70, 300, 1440), (140, 257, 2000), (300, 128, 1024)):
        ops = operands(M, N, K, M + kind)
        close(mb.gemm_fp8(*ops, flags=tune), *ops)
        close(mb.gemm_fp8(*ops, flags=tune | mb.OUT_BF16), *ops)
    assert mb.lib.miori_device_error_poll() == 0


@pytest.mark.parametrize("M,N,K", [(1, 100, 16384), (3, 200, 16385), (70, 130, 16400), (300, 300, 20000)])
def test_long_sums(M, N, K):
    """On both sides of the longest K of the kernel of few rows, and a refusal where it is asked for more."""
    ops = operands(M, N, K, 9)
    close(mb.gemm_fp8(*ops), *ops)
    if K > 16384:
        with pytest.raises(mb.MioriError, match="K up to 16384"):
            mb.gemm_fp8(*ops, flags=1 << 20)


def test_scales_that_are_broadcast():
    """One scale for all of a, or for all of w: strides of zero."""
    a, _, w, _ = operands(40, 300, 500, 10)
    one = torch.full((1, 1), 0.25, device=DEV)
    sa, sw = one.expand(40, blocks(500)), one.expand(blocks(300), blocks(500))
    close(mb.gemm_fp8(a, sa, w, sw), a, sa, w, sw)


def test_gemm_to_memory_past_32_bits():
    """Rows of C that begin more than 2^32 bytes behind the first, by both kernels."""
    for M, N in ((600, 200), (70, 130)):
        a, sa, w, sw = operands(M, N, 256, 11)
        pitch = 2 ** 32 // M // 2 // 8 * 8 + 4096  # bf16
        out = torch.full((M, pitch), 2.0, dtype=torch.bfloat16, device=DEV)
        got = mb.gemm_fp8(a, sa, w, sw, flags=mb.OUT_BF16, out=out[:, :N])
        close(got, a, sa, w, sw)
        assert bool((out[-1, N:] == 2).all()) and bool((out[0, N:] == 2).all())
        del out, got


def test_quant_of_memory_past_32_bits():
    x = torch.zeros((3, 2 ** 30 + 64), dtype=torch.float32, device=DEV)[:, :700]
    x.copy_(torch.randn(3, 700, device=DEV, generator=torch.Generator(device=DEV).manual_seed(12)))
    for tile in (1, 128):
        same(mb.quant_fp8(x, tile=tile), oracle_quant(x, tile))


def test_quant_rows_do_not_depend_on_one_another():
    """A row's codes and scales in blocks of one row are the same alone, in a small and in a large batch (other numbers of lanes a block)."""
    x = torch.randn(5000, 1440, device=DEV, generator=torch.Generator(device=DEV).manual_seed(13))
    q, s = mb.quant_fp8(x)
    for rows in (1, 2, 7, 33, 600):
        part, ps = mb.quant_fp8(x[100:100 + rows])
        assert torch.equal(bits(part), bits(q)[100:100 + rows]) and torch.equal(ps, s[100:100 + rows])
