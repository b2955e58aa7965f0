"""Layers of experts against 64-bit arithmetic.

Tolerance, element by element.  Activations are fp16 times a power of two: x (bf16) without a rounding that shows (2^-27 of the largest of 128), the activation
between the products 2^-11 of a value.  Sums of n products in fp32 by MMAs: what an MMA's 16 products and the running sum lose is at most 17 * 2^-24 of the sum
A of absolute values; (n / 16) of them, and as many additions of partial sums and scales at most: within n * 2^-23 * A, and A is taken of |s| code + |b| where weights
are packed.  That of gate and up goes through silu(g) u, whose slopes are at most 1.1 |u| and |silu(g)|."""
import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP8 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // 128)


def make(bits, group, T, E, H, F, seed, bias=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x = (randn(T, H) * torch.exp(randn(T, 1)) * (0.2 + rand(H))).to(torch.bfloat16)
    router = (randn(E, H) / H ** 0.5).to(torch.bfloat16)
    ws = []
    for N, K in ((2 * F, H), (H, F)):
        if bits == 4:
            s = (0.004 * (0.3 + rand(E, N, K // group))).to(torch.bfloat16)
            ws += [torch.randint(-2 ** 31, 2 ** 31, (E, N, K // 8), generator=g, device=DEV).to(torch.int32), s, (-7.5 * s.float() * (0.8 + 0.4 * rand(s.shape))).to(torch.bfloat16)]
        else:
            ws += [(randn(E, N, K) * 100).clamp(-448, 448).to(FP8), 2e-4 * (0.3 + rand(E, blocks(N), blocks(K)))]
    return x, router, ws, 0.2 * randn(E) if bias else None


def dense(kept, e, bits, group):
    """(W, |W|) of an expert in 64 bits."""
    if bits == 8:
        w, s = kept[0][e].double(), kept[1][e].double()
        w = w * s[torch.arange(w.shape[0], device=DEV) // 128][:, torch.arange(w.shape[1], device=DEV) // 128]
        return w, w.abs()
    words, s, b = (t[e] for t in kept)
    k = torch.arange(words.shape[1] * 8, device=DEV)
    codes, s, b = ((words.long()[:, k // 8] >> (4 * (k % 8))) & 15).double(), s.double()[:, k // group], b.double()[:, k // group]
    return codes * s + b, codes * s.abs() + b.abs()


def choice(x, router, top, bias, sigmoid, norm, factor):
    """[(expert, weight)] of each token."""
    l = x.double() @ router.double().T
    p = torch.sigmoid(l) if sigmoid else torch.softmax(l, 1)
    r = l if bias is None else p + bias.double()
    lists = []
    for t in range(x.shape[0]):
        order = torch.sort(r[t], descending=True, stable=True).indices[:top].tolist()
        order = [e for e in order if r[t, e] != -float("inf") or bias is None]
        w = [float(p[t, e]) for e in order]
        lists.append([(e, v / (sum(w) if norm else 1.0) * factor) for e, v in zip(order, w)])
    return lists


def oracle(x, router, ws, bits, group, top, bias, sigmoid, norm, factor):
    T, H = x.shape
    half = len(ws) // 2
    F = ws[half].shape[2] * (8 if bits == 4 else 1)
    out, tol = (torch.zeros(T, H, dtype=torch.float64, device=DEV) for _ in range(2))
    lists = choice(x, router, top, bias, sigmoid, norm, factor)
    for e in sorted({e for row in lists for e, _ in row}):
        (up, up_abs), (down, down_abs) = dense(ws[:half], e, bits, group), dense(ws[half:], e, bits, group)
        for t, row in enumerate(lists):
            for w in [w for i, w in row if i == e]:
                v = x[t].double()
                gu, room = up @ v, up_abs @ v.abs() * (H * 2.0 ** -23)
                g, u = gu[:F], gu[F:]
                silu = g / (1 + torch.exp(-g))
                h = silu * u
                dh = 1.1 * u.abs() * room[:F] + silu.abs() * room[F:] + h.abs() * 2.0 ** -20
                out[t] += w * (down @ h)
                tol[t] += abs(w) * (down_abs @ (h.abs() * (2.0 ** -11 + F * 2.0 ** -23) + dh + h.abs().max() * 2.0 ** -38))
    return out, tol


def run(x, router, ws, bits, group, top, bias, flags, factor=1.0, workspace=None, out=None):
    F = ws[0].shape[1] // 2
    workspace = mb.moe_workspace(x.shape[0], top, F, DEV) if workspace is None else workspace
    if bits == 4:
        return mb.moe4(x, router, *ws, top, workspace, bias=bias, group=group, factor=factor, flags=flags, out=out)
    return mb.moe_fp8(x, router, *ws, top, workspace, bias=bias, factor=factor, flags=flags, out=out)


def check(x, router, ws, bits, group, top, bias, flags, factor=1.0):
    got = run(x, router, ws, bits, group, top, bias, flags, factor)
    want, tol = oracle(x, router, ws, bits, group, top, bias, bool(flags & mb.MOE_SIGMOID), bool(flags & mb.MOE_NORM), factor)
    if flags & mb.OUT_BF16:
        tol = tol + want.abs() * 2.0 ** -8
    assert got.shape == x.shape
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((got.double() - want).abs() / tol).max()))
    # as a whole: the roundings are of either sign
    assert float((got.double() - want).norm() / want.norm()) < (1e-2 if flags & mb.OUT_BF16 else 2.0 ** -11)
    assert mb.lib.miori_device_error_poll() == 0
    return got


SHAPES = [(1, 32, 4, 2048, 1536), (1, 1, 1, 128, 128), (2, 8, 2, 256, 384), (3, 20, 3, 1408, 640), (4, 64, 8, 2048, 768), (7, 5, 5, 512, 1280), (8, 32, 4, 2048, 1536),
          (9, 8, 2, 1024, 896), (13, 256, 16, 384, 128), (16, 17, 1, 640, 256), (32, 32, 4, 2048, 1536), (32, 2, 2, 256, 512), (31, 40, 6, 4096, 256), (32, 128, 8, 1152, 384)]


@pytest.mark.parametrize("T,E,top,H,F", SHAPES)
@pytest.mark.parametrize("bits,group", [(4, 64), (4, 32), (8, 128)])
def test_layers(T, E, top, H, F, bits, group):
    x, router, ws, bias = make(bits, group, T, E, H, F, T + E + H, bias=T % 2 == 1)
    flags = (mb.MOE_SIGMOID if T % 3 == 1 else 0) | (mb.MOE_NORM if E % 2 == 0 else 0) | (mb.OUT_BF16 if T % 4 == 3 else 0)
    check(x, router, ws, bits, group, top, bias, flags, 1.0 if T != 2 else -2.5)


@pytest.mark.parametrize("T,E,top,H,F", [(1, 4, 2, 16, 16), (5, 20, 3, 1440, 720), (13, 20, 3, 1440, 720), (20, 9, 2, 144, 2064), (32, 33, 4, 3040, 336)])
def test_sizes_that_end_inside_a_block(T, E, top, H, F):
    x, router, ws, bias = make(8, 128, T, E, H, F, T * 3 + E)
    check(x, router, ws, 8, 128, top, bias, mb.MOE_NORM)


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 128)])
def test_all_tokens_choose_the_same_experts(bits, group):
    """Experts of 32 tokens, and none for the others."""
    x, router, ws, _ = make(bits, group, 32, 12, 384, 256, 5)
    bias = torch.full((12,), -10.0, device=DEV)
    bias[3], bias[11] = 10.0, 20.0
    check(x, router, ws, bits, group, 2, bias, mb.MOE_SIGMOID)


def test_experts_that_are_never_chosen():
    """A bias of -inf takes an expert out; with too few left a token has fewer, with none a row of zeros."""
    x, router, ws, bias = make(4, 64, 6, 8, 256, 256, 6)
    bias[[0, 2, 3, 4, 6, 7]] = -float("inf")
    check(x, router, ws, 4, 64, 3, bias, mb.MOE_NORM)
    bias[:] = -float("inf")
    out = torch.full((6, 256), 7.0, device=DEV)
    run(x, router, ws, 4, 64, 3, bias, mb.MOE_NORM, out=out)
    assert not bool(out.any())


def test_equal_scores_go_to_the_lowest_index():
    x, router, ws, _ = make(4, 64, 3, 70, 128, 128, 7)
    router[:] = router[0]
    lists = choice(x, router, 5, None, False, True, 1.0)
    assert all([e for e, _ in row] == [0, 1, 2, 3, 4] for row in lists)
    check(x, router, ws, 4, 64, 5, None, mb.MOE_NORM)


def test_rows_of_zeros_and_of_no_numbers():
    """A token of zeros gives zeros of a sum; one with a NaN or an infinity spoils itself alone."""
    x, router, ws, _ = make(8, 128, 5, 8, 256, 256, 8)
    x[1] = 0.0
    clean = run(x, router, ws, 8, 128, 2, None, 0)
    assert not bool(clean[1].any())
    x[2, 5], x[4, 9] = float("nan"), float("inf")
    got = run(x, router, ws, 8, 128, 2, None, 0)
    assert bool(torch.isnan(got[2]).all()) and not bool(torch.isfinite(got[4]).any())
    # the others: whatever the spoilt rows chose, within the sums' order
    for t in (0, 1, 3):
        torch.testing.assert_close(got[t], clean[t], rtol=0, atol=float(clean[t].abs().max()) * 2.0 ** -18)


@pytest.mark.parametrize("bits,group", [(4, 64), (4, 32), (8, 128)])
def test_activations_of_very_different_sizes(bits, group):
    """An outlier in a block of 128, and blocks far from one another in size."""
    x, router, ws, bias = make(bits, group, 2, 8, 512, 256, 9)
    x = x.float()
    x[0, 77] = 3e4
    x[1, :128] *= 1e-20
    x[1, 256:384] *= 1e-6
    x = x.to(torch.bfloat16)
    router = router * 1e-3
    check(x, router, ws, bits, group, 2, bias, mb.MOE_SIGMOID)


@pytest.mark.parametrize("bits,group,T", [(4, 64, 1), (4, 32, 11), (8, 128, 32)])
def test_repeats_graphs_streams_and_a_workspace_used_again(bits, group, T):
    """The same bits from call to call; a graph replayed with new tokens; a workspace that a larger call has used."""
    x, router, ws, bias = make(bits, group, T, 16, 512, 384, 10)
    workspace = mb.moe_workspace(32, 4, 384, DEV)
    first = run(x, router, ws, bits, group, 4, bias, 0, workspace=workspace)
    more = make(bits, group, 32, 16, 512, 384, 11)[0]
    run(more, router, ws, bits, group, 4, bias, 0, workspace=workspace)
    for _ in range(3):
        assert torch.equal(first, run(x, router, ws, bits, group, 4, bias, 0, workspace=workspace))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own = run(x, router, ws, bits, group, 4, bias, 0)  # a workspace of its own
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, own)
    given = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(given, router, ws, bits, group, 4, bias, 0, workspace=workspace)
        out2 = run(given, router, ws, bits, group, 4, bias, 0, workspace=workspace)
    graph.replay()
    assert torch.equal(first, out) and torch.equal(first, out2)
    given.copy_(more[:T])
    graph.replay()
    assert torch.equal(run(more[:T].contiguous(), router, ws, bits, group, 4, bias, 0, workspace=workspace), out)
    assert mb.lib.miori_device_error_poll() == 0


def test_between_launches_that_may_begin_early():
    """rmsnorm in front and a projection behind, both launched so that they may overlap what is before them."""
    from miori_b200 import synth
    x, router, ws, bias = make(4, 64, 4, 16, 512, 384, 12)
    q, s, b = synth.make_weight(256, 512, 4, 64, seed=4, device=DEV)
    gamma = torch.ones(512, dtype=torch.bfloat16, device=DEV)
    workspace = mb.moe_workspace(4, 2, 384, DEV)
    for i in range(20):
        r = torch.randn(4, 512, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i))
        n = mb.rmsnorm(r, gamma, 1e-5, mb.LAUNCH_PDL)
        y = run(n, router, ws, 4, 64, 2, bias, mb.OUT_BF16 | mb.LAUNCH_PDL, workspace=workspace)
        z = mb.gemv4(q, s, b, y, 64, mb.LAUNCH_PDL)
        torch.cuda.synchronize()
        n2 = mb.rmsnorm(r, gamma, 1e-5)
        torch.cuda.synchronize()
        y2 = run(n2, router, ws, 4, 64, 2, bias, mb.OUT_BF16, workspace=workspace)
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and torch.equal(z, mb.gemv4(q, s, b, y2, 64))


@pytest.mark.parametrize("bits,group,T,E,top,H,F", [
    (4, 64, 3, 4, 2, 7168, 256), (4, 32, 20, 4, 2, 7168, 128), (8, 128, 9, 4, 3, 7168, 144),  # rows whose B fragments take a shorter ring
    (4, 64, 32, 128, 16, 2048, 128), (4, 32, 32, 256, 8, 7168, 128), (8, 128, 32, 256, 16, 1024, 128),  # so many entries that rows of the output are worked on in parts
    (4, 64, 2, 2, 1, 128, 65536), (8, 128, 2, 1, 1, 16, 65536), (8, 128, 32, 3, 2, 16, 16)])
def test_the_largest_and_the_smallest(bits, group, T, E, top, H, F):
    x, router, ws, bias = make(bits, group, T, E, H, F, T + E + 1)
    check(x, router, ws, bits, group, top, bias, mb.MOE_SIGMOID)


@pytest.mark.parametrize("flags", [0, 1 << 10])
def test_logits_far_from_zero(flags):
    """Scores that are one, or underflow: shares of them stay shares.  (Logits of a single product, which fp32 holds: only the exponentials round.)"""
    assert mb.MOE_NORM == 1 << 10
    x, router, ws, bias = make(4, 64, 6, 12, 256, 128, 14)
    column = (router[:, 0].float() * 16 * 60).to(torch.bfloat16)
    router = torch.zeros_like(router)
    router[:, 0] = column
    x[:, 0] = torch.tensor([1.0, -1.0, 0.5, 2.0, -2.0, 0.25], device=DEV).to(torch.bfloat16)
    check(x, router, ws, 4, 64, 3, None, flags)
    check(x, router, ws, 4, 64, 3, None, flags | mb.MOE_SIGMOID)
    # a bias that picks experts whose scores are nothing in fp32; with logits of -200 and so on a 64-bit oracle still has them
    x[:, 0] = 1.0
    low = torch.zeros_like(router)
    low[:, 0] = torch.arange(12, device=DEV) * -2.0 - 200.0
    low[5] = 0.0
    bias = torch.zeros(12, device=DEV)
    bias[[2, 3, 4]] = 5.0
    if flags & mb.MOE_NORM:
        check(x, low, ws, 4, 64, 3, bias, flags)
        check(x, low, ws, 4, 64, 3, bias, flags | mb.MOE_SIGMOID)


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 128)])
def test_in_place(bits, group):
    x, router, ws, bias = make(bits, group, 7, 8, 256, 256, 15)
    want = run(x, router, ws, bits, group, 2, bias, mb.OUT_BF16)
    got = run(x, router, ws, bits, group, 2, bias, mb.OUT_BF16, out=x)
    assert got is x and torch.equal(got, want)


def test_two_streams_at_once():
    """Layers that overlap, each with a workspace of its own."""
    sides, results = [torch.cuda.Stream() for _ in range(2)], [[], []]
    problems = [make(4, 64, 32, 16, 1024, 512, 16), make(8, 128, 5, 16, 1024, 512, 17)]
    want = [run(problems[0][0], *problems[0][1:3], 4, 64, 2, problems[0][3], 0), run(problems[1][0], *problems[1][1:3], 8, 128, 2, problems[1][3], 0)]
    torch.cuda.synchronize()
    spaces = [mb.moe_workspace(32, 2, 512, DEV) for _ in range(2)]
    for _ in range(20):
        for i, (x, router, ws, bias) in enumerate(problems):
            with torch.cuda.stream(sides[i]):
                results[i].append(run(x, router, ws, (4, 8)[i], (64, 128)[i], 2, bias, mb.LAUNCH_PDL, workspace=spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r, want[i]) for r in results[i])
    assert mb.lib.miori_device_error_poll() == 0
