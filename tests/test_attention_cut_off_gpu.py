"""Requests that end beyond the tensors: a table too short for their positions, fewer rows of q than their tokens, fewer keys than
cu_k says.  What is there is computed as if the rest were too: row t of a request sees the first lens - cu[r + 1] + t + 1 positions, of
those that are there.  Rows of no request, and all around the output, stay as they were.

Tolerance as for the operators in general: 2^-8 of sum_j w_j |v_j| and of |o| for the two roundings to bf16, 2^-13 of the former for fp32.
"""
import math

import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LEFT = -77.0  # what lies in and around an output before the call


@pytest.fixture(scope="module")
def workspace():
    return mb.attention_workspace(DEV)


def check_errors():
    torch.cuda.synchronize()
    assert mb.lib.miori_device_error_poll() == 0


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rand(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV).to(torch.bfloat16)


class Framed:
    """An output inside a larger tensor."""

    def __init__(self, T, H, D):
        self.all = torch.full((T + 2, H + 1, D + 8), LEFT, dtype=torch.bfloat16, device=DEV)
        self.out = self.all[1:T + 1, :H, :D]

    def check(self, o, mass, owned):
        frame = self.all.clone()
        frame[1:-1, :self.out.shape[1], :self.out.shape[2]][owned] = LEFT
        assert (frame == LEFT).all(), "written where nothing belongs"
        if not owned.any():
            return
        got = self.out[owned].double()
        assert torch.isfinite(got).all()
        worst = ((got - o[owned]).abs() / (mass[owned] * (2.0 ** -8 + 2.0 ** -13) + o[owned].abs() * 2.0 ** -8 + 1e-30)).max().item()
        assert worst <= 1.0, f"{worst:.2f} times the bound"


def row(q, k, v, sees):
    """One token in 64 bits over the first `sees` positions."""
    H, D = q.shape
    if sees <= 0:
        return torch.zeros(H, D, dtype=torch.float64, device=DEV), torch.zeros(H, D, dtype=torch.float64, device=DEV)
    k, v = (t[:sees].double().repeat_interleave(H // t.shape[1], 1) for t in (k, v))
    w = torch.softmax(torch.einsum("hd,lhd->hl", q.double(), k) / math.sqrt(D), -1)
    return torch.einsum("hl,lhd->hd", w, v), torch.einsum("hl,lhd->hd", w, v.abs())


def expected(q, cu, lens, keys, causal=True):
    """keys[r]: what is there of request r's keys and values."""
    T, H, D = q.shape
    o, mass = torch.zeros(T, H, D, dtype=torch.float64, device=DEV), torch.zeros(T, H, D, dtype=torch.float64, device=DEV)
    owned = torch.zeros(T, dtype=torch.bool, device=DEV)
    for r, (k, v) in enumerate(keys):
        for t in range(max(cu[r], 0), min(cu[r + 1], T)):
            owned[t] = True
            o[t], mass[t] = row(q[t], k, v, min(max(lens[r], 0) - cu[r + 1] + t + 1, k.shape[0]) if causal else k.shape[0])
    return o, mass, owned


def paged(seed, T, cu, lens, width, H, G, D, page, said, workspace, causal=True, garbage=math.nan):
    """Positions that nobody has written (behind the rows that are there) hold `garbage`."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    R = len(lens)
    table = torch.randperm(R * width + 1, generator=g, device=DEV)[:R * width].view(R, width)
    cache = torch.full((2, R * width + 1, G, page, D), garbage, dtype=torch.bfloat16, device=DEV)
    q, keys = rand(g, T, H, D), []
    for r in range(R):
        L = max(0, min(lens[r], width * page))
        kv, p = rand(g, 2, L, G, D), torch.arange(L, device=DEV)
        written = L if not causal else min(L, max(0, lens[r] - max(0, cu[r + 1] - T)))
        for i in range(2):
            cache[i][table[r, p[:written] // page], :, p[:written] % page] = kv[i, :written]
        keys.append((kv[0], kv[1]))
    f = Framed(T, H, D)
    mb.attention_paged(q, cache[0], cache[1], table.to(torch.int32), i32(lens), i32(cu), said, out=f.out, workspace=workspace,
                       flags=0 if causal else mb.ATTENTION_FULL)
    check_errors()
    f.check(*expected(q, cu, lens, keys, causal))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("said", [1, 1000])
@pytest.mark.parametrize("shared", [True, False])
def test_a_table_that_is_too_short(D, said, shared, workspace):
    ws = workspace if shared else None
    paged(1, 42, [0, 40, 42], [70, 40], 3, 8, 2, D, 16, said, ws)           # 70 positions, 48 of them in the table
    paged(2, 6, [0, 1, 4, 6], [49, 500, 30], 3, 8, 2, D, 16, said, ws)      # some tokens stand behind what is there
    paged(3, 300, [0, 290, 300], [700, 700], 16, 4, 1, D, 32, said, ws)     # many items, the last ones behind it
    paged(4, 300, [0, 290, 300], [700, 100], 16, 4, 1, D, 32, said, ws, causal=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("said", [1, 1000])
@pytest.mark.parametrize("garbage", [math.nan, math.inf, 3.0e38])
def test_fewer_rows_than_tokens(D, said, garbage, workspace):
    paged(5, 25, [0, 40], [70], 6, 8, 2, D, 16, said, workspace, garbage=garbage)
    paged(6, 1, [0, 4], [70], 6, 8, 2, D, 16, said, workspace, garbage=garbage)      # one row, and positions that it does not see
    paged(7, 9, [0, 5, 300], [5, 420], 30, 8, 2, D, 16, said, workspace, garbage=garbage)
    paged(8, 200, [0, 150, 2 ** 31 - 1], [150, 2 ** 31 - 1], 30, 4, 2, D, 16, said, workspace, garbage=garbage)
    paged(9, 200, [0, 150, 400], [100, 240], 30, 4, 2, D, 16, said, workspace, garbage=garbage)  # and fewer positions than tokens


@pytest.mark.parametrize("said", [1, 1000])
@pytest.mark.parametrize("cu", [[0, 3, 6], [0, 100, 2 ** 31 - 1], [-4, 2, -1], [5, 2, 9], [1, 1, 4], [7, 8, 9]])
@pytest.mark.parametrize("lens", [[48, 20], [1000, -5], [2 ** 31 - 1, 48], [0, 7]])
def test_odd_numbers(cu, lens, said, workspace):
    paged(10, 6, cu, lens, 3, 4, 2, 64, 16, said, workspace, garbage=0.5)
    paged(11, 6, cu, lens, 3, 4, 2, 128, 8, said, None, garbage=0.5)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,keys,cu,cu_k", [
    (50, 50, [0, 70], None),                    # rows of q and of keys end inside the only prompt
    (50, 70, [0, 70], [0, 70]),                 # rows of q only
    (70, 50, [0, 70], [0, 70]),                 # keys only
    (90, 60, [0, 20, 100], [0, 30, 120]),
    (700, 700, [0, 30, 900], None), (700, 900, [0, 30, 900], [0, 30, 900]), (900, 600, [0, 30, 900], [0, 30, 900]),
    (600, 10, [0, 700], [0, 700]), (600, 600, [-3, 700], [-5, 600]), (600, 600, [0, 2 ** 31 - 1], [0, 2 ** 31 - 1])])
@pytest.mark.parametrize("shared", [True, False])
def test_packed_prompts(D, T, keys, cu, cu_k, shared, workspace):
    g = torch.Generator(device=DEV).manual_seed(12)
    H, G = 4, 2
    q, k, v = rand(g, T, H, D), rand(g, keys, G, D), rand(g, keys, G, D)
    ck = [max(c, 0) for c in (cu if cu_k is None else cu_k)]
    there = [(k[a:min(b, keys)], v[a:min(b, keys)]) for a, b in zip(ck, ck[1:])]
    f = Framed(T, H, D)
    mb.attention_prompt(q, k, v, i32(cu), cu_k=None if cu_k is None else i32(cu_k), out=f.out, workspace=workspace if shared else None)
    check_errors()
    f.check(*expected(q, cu, [b - a for a, b in zip(ck, ck[1:])], there))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("width,rows", [(3, 45), (6, 22), (2, 30)])
@pytest.mark.parametrize("said", [1, 1000])
def test_a_step_cut_off_by_page_slots(D, width, rows, said, workspace):
    """Held 30, 40 new, and 5 beside them, in a table or with rows that are too short: whoever got a slot is computed right."""
    page, H, G, held, new = 16, 4, 1, [30, 0], [40, 5]
    g = torch.Generator(device=DEV).manual_seed(13)
    table = i32([[3, 4] + [-1] * (width - 2), [-1] * width])
    slots, positions, cu, lens, _ = mb.page_slots(i32(held), i32(new), table, i32([0, 1, 2, 5, 6, 7]), i32([0]), page, rows)
    qkv = torch.randn(rows, (H + 2 * G) * D, generator=g, device=DEV)
    cache = torch.full((2, 8, G, page, D), math.nan, dtype=torch.bfloat16, device=DEV)
    cache[:, 3:5] = rand(g, 2, 2, G, page, D)
    turns, axes = mb.rope_turns(D, theta=1e4, device=DEV)
    q = mb.rope_kv(qkv, turns, positions, slots, cache[0], cache[1], H, axes=axes)
    f = Framed(rows, H, D)
    mb.attention_paged(q, cache[0], cache[1], table, lens, cu, said, out=f.out, workspace=workspace)
    check_errors()
    keys = []
    for r, n in enumerate(lens.tolist()):
        p = torch.arange(min(n, width * page), device=DEV)
        numbers = table[r].long()[p // page].clamp(min=0)
        keys.append(tuple(c[numbers, :, p % page] for c in cache))
    o, mass, owned = expected(q, cu.tolist(), lens.tolist(), keys)
    assert bool(owned.all()) == (rows <= 45)
    f.check(o, mass, owned)
