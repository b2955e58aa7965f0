"""Attention over the page cache and over packed prompts, against the formula in 64 bits.

Tolerance, from the formula.  With probabilities w (sum 1), the kernel rounds each p to bf16 once and the result once; bf16 has
eight significant bits, so each rounding is off by up to 2^-8 of its value (1 + 2^-8 lies halfway between two numbers).
Everything else is fp32 with sums of at most 2^15 terms (2^-24 each, and 2^-21 for the exponential of a score of up to 16):
|error| <= 2^-8 * sum_j w_j |v_j| + 2^-8 * |o| + 2^-13 * sum_j w_j |v_j|.
"""
import math

import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def workspace():
    return mb.attention_workspace(DEV)


def check_errors():
    torch.cuda.synchronize()
    assert mb.lib.miori_device_error_poll() == 0


def formula(q, k, v, first, causal=True, scale=None):
    """One request in 64 bits: q [n][H][D], whose token i sees the first `first` + i + 1 rows of k and v [L][G][D].
    Returns o and sum_j w_j |v_j|; rows that see nothing are zeros."""
    n, H, D = q.shape
    L, G = k.shape[:2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o, mass = torch.zeros(n, H, D, dtype=torch.float64, device=q.device), torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    for i in range(n):
        sees = min(L, first + i + 1) if causal else L
        if sees <= 0:
            continue
        kk, vv = k[:sees].double().repeat_interleave(H // G, 1), v[:sees].double().repeat_interleave(H // G, 1)
        w = torch.softmax(torch.einsum("hd,lhd->hl", q[i].double(), kk) * scale, -1)
        o[i] = torch.einsum("hl,lhd->hd", w, vv)
        mass[i] = torch.einsum("hl,lhd->hd", w, vv.abs())
    return o, mass


def formula_fast(q, k, v, first, causal=True, scale=None):
    """The same for requests too long to go token by token (every token sees a position, values are finite)."""
    n, H, D = q.shape
    L, G = k.shape[:2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o, mass = torch.empty(n, H, D, dtype=torch.float64, device=q.device), torch.empty(n, H, D, dtype=torch.float64, device=q.device)
    hidden = torch.arange(L, device=q.device)[None] > first + torch.arange(n, device=q.device)[:, None]
    for h in range(H):
        x = q[:, h].double() @ k[:, h // (H // G)].double().T * scale
        w = torch.softmax(x.masked_fill(hidden, -math.inf) if causal else x, -1)
        o[:, h], mass[:, h] = w @ v[:, h // (H // G)].double(), w @ v[:, h // (H // G)].double().abs()
    return o, mass


def assert_near(got, o, mass, what=""):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bound = mass * (2.0 ** -8 + 2.0 ** -13) + o.abs() * 2.0 ** -8 + 1e-30
    worst = ((got - o).abs() / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound"


def rand(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(torch.bfloat16)


def cu_of(lengths):
    return torch.tensor([0] + lengths, device=DEV).cumsum(0).to(torch.int32)


# ---- packed prompts -----------------------------------------------------------------------

def prompt_case(seed, lengths, H, G, D, workspace, keys=None, causal=True, scale=None, qs=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    keys = lengths if keys is None else keys
    q, k, v = rand(g, sum(lengths), H, D, scale=qs), rand(g, sum(keys), G, D), rand(g, sum(keys), G, D)
    out = mb.attention_prompt(q, k, v, cu_of(lengths), cu_k=None if keys is lengths else cu_of(keys), scale=scale,
                              flags=0 if causal else mb.ATTENTION_FULL, workspace=workspace)
    check_errors()
    a = b = 0
    for n, L in zip(lengths, keys):
        if n:
            f = formula if n <= 40 or L < n else formula_fast
            assert_near(out[a:a + n], *f(q[a:a + n], k[b:b + L], v[b:b + L], L - n, causal, scale), f"prompt of {n}, {L} keys")
        a, b = a + n, b + L
    return out


@pytest.mark.parametrize("H,G,D", [(16, 4, 128), (8, 8, 128), (4, 1, 64), (15, 5, 128), (14, 2, 64), (12, 4, 128), (64, 1, 64), (7, 1, 128)])
@pytest.mark.parametrize("lengths", [[1], [77], [128], [129, 1, 300], [0, 5, 0, 64, 63, 65, 0]])
@pytest.mark.parametrize("shared", [True, False])
def test_prompts(H, G, D, lengths, shared, workspace):
    prompt_case(1, lengths, H, G, D, workspace if shared else None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[1500], [2047, 3, 700], [31] * 33, [1023, 1025]])
@pytest.mark.parametrize("causal", [True, False])
def test_longer_prompts(D, lengths, causal, workspace):
    prompt_case(2, lengths, 8, 2, D, workspace, causal=causal)


@pytest.mark.parametrize("H,G,D", [(16, 4, 128), (8, 8, 128), (4, 1, 64), (15, 5, 128), (14, 2, 64), (12, 4, 128), (64, 1, 64), (7, 1, 128)])
@pytest.mark.parametrize("lengths", [[1, 600], [77, 512], [700, 128], [129, 1, 300, 211], [0, 5, 0, 64, 777, 63, 65, 0]])
@pytest.mark.parametrize("shared", [True, False])
def test_prompts_beside_long_ones(H, G, D, lengths, shared, workspace):
    """Odd lengths among so many tokens that the tensor-memory kernel takes them."""
    prompt_case(31, lengths, H, G, D, workspace if shared else None)


@pytest.mark.parametrize("D", [64, 128])
def test_many_short_prompts(D, workspace):
    prompt_case(32, [(i * 5) % 67 for i in range(60)], 8, 2, D, workspace)
    prompt_case(33, [60] * 34, 8, 2, D, workspace, causal=False)


@pytest.mark.parametrize("tokens,keys", [([700, 3], [9, 600]), ([40, 800], [1, 1]), ([600, 10], [0, 400]), ([3, 650], [2000, 650])])
@pytest.mark.parametrize("causal", [True, False])
def test_many_keys_of_their_own(tokens, keys, causal, workspace):
    prompt_case(34, tokens, 4, 2, 64, workspace, keys=keys, causal=causal)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("at", [599, 640, 700, 701])
def test_what_a_token_of_a_long_prompt_does_not_see(bad, at, workspace):
    """As below, in the tensor-memory kernel: a value that is not finite reaches exactly the tokens that see it, in its dimensions."""
    g = torch.Generator(device=DEV).manual_seed(35)
    lengths, H, G, D = [701, 150], 4, 2, 128
    q, k, v = rand(g, 851, H, D), rand(g, 851, G, D), rand(g, 851, G, D)
    clean = mb.attention_prompt(q, k, v, cu_of(lengths), workspace=workspace)
    v[at, 1, 3::5] = bad
    got = mb.attention_prompt(q, k, v, cu_of(lengths), workspace=workspace)
    check_errors()
    hit = torch.zeros(851, H, D, dtype=torch.bool, device=DEV)
    hit[at:(701 if at < 701 else 851), H // 2:, 3::5] = True
    assert torch.equal(got[~hit], clean[~hit])
    assert (torch.isnan(got[hit].float()) if bad != bad else got[hit].float() == bad).all()


def test_more_requests_than_a_warp(workspace):
    prompt_case(3, [(i * 7) % 23 for i in range(300)], 4, 2, 64, workspace)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("tokens,keys", [([5, 3, 200], [9, 1, 60]), ([40], [1]), ([3, 2], [0, 400]), ([10, 10], [300, 0]), ([1], [5000])])
def test_keys_of_their_own(tokens, keys, causal, workspace):
    """More tokens than keys: the first ones see none and get zeros; a request without keys too."""
    prompt_case(4, tokens, 4, 2, 128, workspace, keys=keys, causal=causal)


def test_large_scores_and_other_scales(workspace):
    """Running maxima that move a lot: scores of up to some hundreds, and a scale of one's own."""
    prompt_case(5, [700], 8, 2, 128, workspace, qs=8.0)
    prompt_case(6, [700], 8, 2, 64, workspace, scale=1.7)
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, v = rand(g, 600, 4, 128), rand(g, 600, 2, 128), rand(g, 600, 2, 128)
    k = (k.float() * torch.linspace(0.01, 6.0, 600, device=DEV)[:, None, None]).to(torch.bfloat16)  # ever larger
    out = mb.attention_prompt(q, k, v, cu_of([600]), workspace=workspace)
    assert_near(out, *formula_fast(q, k, v, 0))


def test_strided_views_and_outputs(workspace):
    """q, k and v as views of one projection's rows; an output inside a larger tensor."""
    g = torch.Generator(device=DEV).manual_seed(8)
    H, G, D, T = 8, 2, 128, 210
    qkv = rand(g, T, (H + 2 * G) * D)
    q, k, v = (x.view(T, -1, D) for x in qkv.split([H * D, G * D, G * D], 1))
    big = torch.full((T, H + 3, D + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    out = big[:, 1:H + 1, :D]
    got = mb.attention_prompt(q, k, v, cu_of([T]), out=out, workspace=workspace)
    assert got is out
    assert_near(out, *formula_fast(q, k, v, 0))
    rest = big.clone()
    rest[:, 1:H + 1, :D] = 7.0
    assert (rest == 7.0).all()  # nothing beside the output is written
    # heads outside, tokens inside
    q2 = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(mb.attention_prompt(q2, k, v, cu_of([T]), workspace=workspace), out.contiguous())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["next prompt", "later token"])
@pytest.mark.parametrize("which", ["k", "v"])
def test_what_a_token_does_not_see_does_not_reach_it(bad, where, which, workspace):
    g = torch.Generator(device=DEV).manual_seed(9)
    lengths, H, G, D = [150, 70], 4, 2, 128
    q, k, v = rand(g, 220, H, D), rand(g, 220, G, D), rand(g, 220, G, D)
    clean = mb.attention_prompt(q, k, v, cu_of(lengths), workspace=workspace)
    x = k if which == "k" else v
    at = 150 if where == "next prompt" else 140
    x[at, 1, 3::5] = bad
    got = mb.attention_prompt(q, k, v, cu_of(lengths), workspace=workspace)
    check_errors()
    hit = torch.zeros(220, H, dtype=torch.bool, device=DEV)
    hit[at:(220 if where == "next prompt" else 150), H // 2:] = True
    assert torch.equal(got[~hit], clean[~hit])
    if which == "v":  # and where it is seen it shows, in its own dimensions
        seen = got[hit].float()
        assert (~torch.isfinite(seen[:, 3::5])).all()
        if bad == bad:
            assert (seen[:, 3::5] == bad).all()
        rest = torch.ones(D, dtype=torch.bool, device=DEV)
        rest[3::5] = False
        assert torch.equal(got[hit][:, rest], clean[hit][:, rest])
    elif bad != bad:
        assert torch.isnan(got[hit].float()).all()


# ---- the page cache -------------------------------------------------------------------------

def paged_case(seed, held, new, H, G, D, page, workspace, max_new=None, garbage=math.nan, causal=True, nhd=False, qs=1.0):
    """Requests of held + new positions; what is not theirs in the cache is `garbage`."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = [a + b for a, b in zip(held, new)]
    owned = [-(-n // page) for n in lens]
    total = sum(owned) + 3
    order = torch.randperm(total, generator=g, device=DEV).tolist()
    shape = (2, total, page, G, D) if nhd else (2, total, G, page, D)
    cache = torch.full(shape, garbage, dtype=torch.bfloat16, device=DEV)
    if nhd:
        cache = cache.transpose(2, 3)
    table = torch.full((len(held), max(owned + [1]) + 1), -1, dtype=torch.int32, device=DEV)
    q = rand(g, sum(new), H, D, scale=qs)
    rows, at = [], 0
    for r, L in enumerate(lens):
        pages = torch.tensor(order[at:at + owned[r]], device=DEV, dtype=torch.long)
        at += owned[r]
        table[r, :owned[r]] = pages.to(torch.int32)
        kv = rand(g, 2, L, G, D)
        rows.append(kv)
        p = torch.arange(L, device=DEV)
        for i in range(2):
            cache[i][pages[p // page], :, p % page] = kv[i]
    cu, ln = cu_of(new), torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = mb.attention_paged(q, cache[0], cache[1], table, ln, cu, max(new) if max_new is None else max_new,
                             flags=0 if causal else mb.ATTENTION_FULL, workspace=workspace)
    check_errors()
    a = 0
    for r, n in enumerate(new):
        if n:
            f = formula if n <= 40 and lens[r] < 4000 else formula_fast
            assert_near(out[a:a + n], *f(q[a:a + n], rows[r][0], rows[r][1], lens[r] - n, causal), f"request {r}: {n} new, {lens[r]} positions")
        a += n
    return out, (q, cache, table, ln, cu)


@pytest.mark.parametrize("H,G,D", [(16, 4, 128), (8, 8, 128), (16, 1, 128), (15, 5, 64), (28, 4, 128), (32, 8, 64), (9, 1, 64)])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("shared", [True, False])
def test_decode(H, G, D, page, shared, workspace):
    paged_case(11, [0, 1, 7, 15, 16, 127, 128, 300, 1000], [1] * 9, H, G, D, page, workspace if shared else None)


@pytest.mark.parametrize("held", [[0], [3000], [20000, 1], [5] * 70])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_lengths(held, D, workspace):
    paged_case(12, held, [1] * len(held), 8, 2, D, 16, workspace)


@pytest.mark.parametrize("H,G", [(8, 2), (8, 8), (3, 1), (4, 1)])
@pytest.mark.parametrize("max_new", [None, 1, 1000])
def test_few_and_many_new_tokens(H, G, max_new, workspace):
    """Whatever is said of the number of new tokens, the results are those of the formula; requests without any are fine."""
    for D in (64, 128):
        paged_case(13, [100, 0, 333, 40, 5], [3, 4, 0, 2, 1], H, G, D, 16, workspace, max_new=max_new)
        paged_case(14, [90, 700], [20, 1], H, G, D, 32, workspace, max_new=max_new)


@pytest.mark.parametrize("page", [8, 32, 128, 512])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shared", [True, False])
def test_chunks(page, D, shared, workspace):
    paged_case(15, [0, 1000, 64, 3], [200, 130, 1, 64], 8, 2, D, page, workspace if shared else None)


@pytest.mark.parametrize("H,G", [(6, 2), (5, 1), (7, 1), (16, 16)])
def test_chunks_of_other_groups(H, G, workspace):
    paged_case(16, [50, 500], [100, 65], H, G, 128, 16, workspace)


def test_long_cache_one_chunk(workspace):
    paged_case(17, [9000], [64], 8, 2, 128, 64, workspace)
    paged_case(18, [9000], [5], 32, 2, 64, 64, workspace)


@pytest.mark.parametrize("new", [1, 3, 70])
def test_cache_in_another_order(new, workspace):
    """Heads inside positions: strides other than the usual ones."""
    paged_case(19, [200, 31], [new, new], 8, 4, 128, 16, workspace, nhd=True)


@pytest.mark.parametrize("new", [1, 3, 70])
def test_all_positions_seen(new, workspace):
    paged_case(20, [200, 31], [new, new], 8, 4, 64, 16, workspace, causal=False)


@pytest.mark.parametrize("new", [2, 4, 40])
@pytest.mark.parametrize("garbage", [math.nan, math.inf, 3.0e38])
def test_fewer_positions_than_tokens(new, garbage, workspace):
    """Lengths shorter than the number of new tokens: the first of them see nothing and get zeros."""
    q = rand(torch.Generator(device=DEV).manual_seed(21), new, 4, 64)
    cache = torch.full((2, 4, 1, 16, 64), garbage, dtype=torch.bfloat16, device=DEV)
    kv = rand(torch.Generator(device=DEV).manual_seed(22), 2, new - 1, 1, 64)
    p = torch.arange(new - 1, device=DEV)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    for i in range(2):
        cache[i][table[0].long()[p // 16], :, p % 16] = kv[i]
    out = mb.attention_paged(q, cache[0], cache[1], table, torch.tensor([new - 1], dtype=torch.int32, device=DEV), cu_of([new]), new, workspace=workspace)
    check_errors()
    assert (out[0] == 0).all()
    assert_near(out, *formula(q, kv[0], kv[1], -1))


@pytest.mark.parametrize("new,held", [(3, 200), (4, 0), (4, 13), (50, 100)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_later_tokens_do_not_reach_earlier_ones(new, held, bad, workspace):
    clean, (q, cache, table, ln, cu) = paged_case(23, [held], [new], 8, 2, 128, 16, workspace)
    p = held + new - 2  # the last token but one
    cache[1][table[0, p // 16].long(), 1, p % 16, 10:20] = bad
    got = mb.attention_paged(q, cache[0], cache[1], table, ln, cu, new, workspace=workspace)
    check_errors()
    assert torch.equal(got[:new - 2], clean[:new - 2]) and torch.equal(got[:, :4], clean[:, :4])
    seen = got[new - 2:, 4:].float()
    assert (torch.isnan(seen[..., 10:20]) if bad != bad else seen[..., 10:20] == bad).all()
    assert torch.equal(seen[..., :10], clean[new - 2:, 4:, :10].float())


def test_results_do_not_change_from_launch_to_launch(workspace):
    """Also right behind one another, and the workspace is left as it was found."""
    for held, new in (([20000, 300, 5], [1, 1, 1]), ([6000, 40], [90, 200])):
        out, (q, cache, table, ln, cu) = paged_case(24, held, new, 8, 2, 128, 16, workspace)
        for _ in range(20):
            assert torch.equal(mb.attention_paged(q, cache[0], cache[1], table, ln, cu, max(new), workspace=workspace), out)
    assert int(workspace[:4096].max()) == 0


def test_other_stream_graph_and_early_start():
    held, new = [3000, 77], [1, 1]
    ws = mb.attention_workspace(DEV)
    out, (q, cache, table, ln, cu) = paged_case(25, held, new, 8, 2, 128, 16, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = mb.attention_paged(q, cache[0], cache[1], table, ln, cu, 1, workspace=ws)
    side.synchronize()
    assert torch.equal(again, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mid = mb.attention_paged(q, cache[0], cache[1], table, ln, cu, 1, flags=mb.LAUNCH_PDL, workspace=ws)
        late = mb.attention_paged(mid, cache[0], cache[1], table, ln, cu, 1, flags=mb.LAUNCH_PDL, workspace=ws)
        wide = mb.attention_paged(late, cache[0], cache[1], table, ln, cu, 100, flags=mb.LAUNCH_PDL, workspace=ws)
    ln -= 5  # lengths are read when the graph runs
    graph.replay()
    check_errors()
    a = mb.attention_paged(q, cache[0], cache[1], table, ln, cu, 1, workspace=ws)
    b = mb.attention_paged(a, cache[0], cache[1], table, ln, cu, 1, workspace=ws)
    c = mb.attention_paged(b, cache[0], cache[1], table, ln, cu, 100, workspace=ws)
    assert torch.equal(mid, a) and torch.equal(late, b) and torch.equal(wide, c)


def test_pages_beyond_32_bits(workspace):
    """A cache of more than 2^32 bytes and elements per tensor: pages at its end are read as those at its start."""
    page, G, D = 128, 2, 128
    pages = (1 << 32) // (page * G * D) + 40  # 2^32 elements and some
    k = torch.empty(pages, G, page, D, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    g = torch.Generator(device=DEV).manual_seed(26)
    last = [pages - 1, 3, pages - 7]
    kv = rand(g, 2, 3 * page, G, D)
    for i, p in enumerate(last):
        k[p], v[p] = (x[i * page:(i + 1) * page].transpose(0, 1) for x in kv)
    table = torch.tensor([last], dtype=torch.int32, device=DEV)
    for new in (1, 33):
        q = rand(g, new, 4, D)
        out = mb.attention_paged(q, k, v, table, torch.tensor([3 * page - 2], dtype=torch.int32, device=DEV), cu_of([new]), new, workspace=workspace)
        check_errors()
        assert_near(out, *formula(q, kv[0][:3 * page - 2], kv[1][:3 * page - 2], 3 * page - 2 - new))


# ---- refusals ---------------------------------------------------------------------------------

def test_refusals(workspace):
    b = dict(dtype=torch.bfloat16, device=DEV)
    q, k, cu = torch.zeros(4, 4, 64, **b), torch.zeros(4, 2, 64, **b), cu_of([4])
    cache = torch.zeros(3, 2, 16, 64, **b)
    table, lens = torch.zeros(1, 3, dtype=torch.int32, device=DEV), cu_of([4])[1:]
    with pytest.raises(TypeError, match="bf16"):
        mb.attention_prompt(q.float(), k, k, cu)
    with pytest.raises(ValueError, match="4 rows expected"):
        mb.attention_prompt(q, k[:3], k[:3], cu)
    with pytest.raises(ValueError, match="differ in size"):
        mb.attention_prompt(q, torch.zeros(4, 2, 128, **b), torch.zeros(4, 2, 128, **b), cu)
    with pytest.raises(TypeError, match="int32"):
        mb.attention_prompt(q, k, k, cu.long())
    with pytest.raises(ValueError, match="last dimension"):
        mb.attention_prompt(torch.zeros(4, 64, 4, **b).transpose(1, 2), k, k, cu)
    with pytest.raises(ValueError, match="shape of q"):
        mb.attention_prompt(q, k, k, cu, out=q[:2])
    with pytest.raises(mb.MioriError, match="64 or 128"):
        mb.attention_prompt(torch.zeros(4, 4, 96, **b), torch.zeros(4, 2, 96, **b), torch.zeros(4, 2, 96, **b), cu)
    with pytest.raises(mb.MioriError, match="evenly"):
        mb.attention_prompt(torch.zeros(4, 5, 64, **b), k, k, cu)
    with pytest.raises(mb.MioriError, match="at most 64"):
        mb.attention_prompt(torch.zeros(4, 65, 64, **b), k[:, :1], k[:, :1], cu)
    with pytest.raises(mb.MioriError, match="positive and finite"):
        mb.attention_prompt(q, k, k, cu, scale=0.0)
    with pytest.raises(mb.MioriError, match="multiples of 8"):
        mb.attention_prompt(torch.zeros(4, 4, 68, **b)[..., :64], k, k, cu)
    with pytest.raises(mb.MioriError, match="multiples of 8"):
        mb.attention_prompt(q, k[:, :1].expand(4, 2, 64), k, cu)
    with pytest.raises(mb.MioriError, match="workspace of"):
        mb.attention_prompt(q, k, k, cu, workspace=workspace[:4096])
    with pytest.raises(mb.MioriError, match="power of two"):
        mb.attention_paged(q, cache[:, :, :12], cache[:, :, :12], table, lens, cu, 4)
    with pytest.raises(mb.MioriError, match="power of two"):
        mb.attention_paged(q, cache[:, :, :4], cache[:, :, :4], table, lens, cu, 4)
    with pytest.raises(ValueError, match="table"):
        mb.attention_paged(q, cache, cache, table[0], lens, cu, 4)
    with pytest.raises(ValueError, match="2 numbers expected"):
        mb.attention_paged(q, cache, cache, table, lens, cu[:1], 4)
    with pytest.raises(ValueError, match="differ in shape"):
        mb.attention_paged(q, cache, cache[:2], table, lens, cu, 4)
    with pytest.raises(mb.MioriError, match="empty shape"):
        mb.attention_paged(q[:0], cache, cache, table, lens, cu, 4)
    check_errors()


def test_lengths_that_contradict_the_tensors(workspace):
    """Nothing beyond the tensors is read or written: lengths and page numbers are cut off."""
    b = dict(dtype=torch.bfloat16, device=DEV)
    q = torch.randn(6, 4, 64, device=DEV).to(torch.bfloat16)
    cache = torch.randn(3, 2, 16, 64, device=DEV).to(torch.bfloat16)
    table = torch.tensor([[1, -1, 10 ** 9], [2, 0, 7]], dtype=torch.int32, device=DEV)
    for new in (1, 50):
        for lens in ([1000, -5], [2 ** 31 - 1, 48], [20, 20]):
            for cu in ([0, 3, 6], [0, 100, 2 ** 31 - 1], [-4, 2, -1], [5, 2, 9]):
                mb.attention_paged(q, cache, cache, table, torch.tensor(lens, dtype=torch.int32, device=DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), new,
                                   workspace=workspace)
    k = torch.zeros(6, 2, 64, **b)
    for cu in ([0, 3, 6], [0, 100, 2 ** 31 - 1], [-4, 2, -1], [5, 2, 9]):
        mb.attention_prompt(q, k, k, torch.tensor(cu, dtype=torch.int32, device=DEV), workspace=workspace)
    check_errors()
    assert int(workspace[:4096].max()) == 0
