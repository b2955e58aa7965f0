"""Positions whose table entry is no page of the cache: no token sees them, in whichever kernel takes the call.

The formula in 64 bits runs over the other positions.  Tolerance as for the operator in general: probabilities are rounded to bf16
once and the result once (2^-8 each, of sum_j w_j |v_j| and of |o|), everything else is fp32 (2^-13 of sum_j w_j |v_j|).
"""
import math

import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NO_PAGE = (-1, -2 ** 31, 10 ** 9, 2 ** 31 - 1)


@pytest.fixture(scope="module")
def workspace():
    return mb.attention_workspace(DEV)


def check_errors():
    torch.cuda.synchronize()
    assert mb.lib.miori_device_error_poll() == 0


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def formula(q, k, v, seen):
    """q [n][H][D], k and v [L][G][D] in 64 bits, seen [n][L]: which positions each token sees."""
    n, H, D = q.shape
    k, v = (t.double().repeat_interleave(H // t.shape[1], 1) for t in (k, v))
    x = torch.einsum("nhd,lhd->nhl", q.double(), k) / math.sqrt(D)
    x = x.masked_fill(~seen[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    w = torch.where(seen[:, None], torch.exp(x - torch.where(torch.isinf(top), 0.0, top)), 0.0)
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
    return torch.einsum("nhl,lhd->nhd", w, v), torch.einsum("nhl,lhd->nhd", w, v.abs())


def assert_near(got, o, mass, what):
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bound = mass * (2.0 ** -8 + 2.0 ** -13) + o.abs() * 2.0 ** -8 + 1e-30
    worst = ((got.double() - o).abs() / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound"


def missing(kind, owned):
    """Which of a request's pages are not there."""
    return {"none": [], "all": range(owned), "first": range(min(1, owned)), "tail": range(owned // 2, owned),
            "some": [i for i in range(owned) if i % 3 == 1 or i % 11 == 4]}[kind]


class Case:
    """Requests of `lens` positions, `new` of them new, some of whose pages are not there."""

    def __init__(self, seed, lens, new, kinds, H, G, D, page):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.page, self.lens, self.new = page, lens, new
        owned = [-(-n // page) for n in lens]
        total, width = sum(owned) + 2, max(owned) + 1
        order = torch.randperm(total, generator=g, device=DEV).tolist()
        self.q, self.cache = (torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16) for s in ((sum(new), H, D), (2, total, G, page, D)))
        self.table, self.there, at = torch.full((len(lens), width), -1, dtype=torch.int32), [], 0
        for r, n in enumerate(owned):
            self.table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
            gone = list(missing(kinds[r], n))
            for i in gone:
                self.table[r, i] = NO_PAGE[i % 4] if i % 5 else total  # the first number that is no page any more
            there = torch.ones(n * page, dtype=torch.bool, device=DEV)
            for i in gone:
                there[i * page:(i + 1) * page] = False
            self.there.append(there[:lens[r]])
        self.table = self.table.to(DEV)
        self.cu = i32([0] + new).cumsum(0).to(torch.int32)

    def run(self, max_new, workspace, cache=None, flags=0):
        cache = self.cache if cache is None else cache
        return mb.attention_paged(self.q, cache[0], cache[1], self.table, i32(self.lens), self.cu, max_new, flags=flags, workspace=workspace)

    def full_table(self):
        """The same requests with a page for every position."""
        t = self.table.clone()
        t[(t < 0) | (t >= self.cache.shape[1])] = 0
        return t

    def check(self, out, causal=True):
        a = 0
        for r, (n, L) in enumerate(zip(self.new, self.lens)):
            p = torch.arange(L, device=DEV)
            numbers = self.table[r].long()[p // self.page]
            numbers = torch.where(self.there[r], numbers, 0)
            k, v = (c[numbers, :, p % self.page] for c in self.cache)
            seen = self.there[r][None].expand(n, L).clone()
            if causal:
                seen &= p[None] < L - n + 1 + torch.arange(n, device=DEV)[:, None]
            o, mass = formula(self.q[a:a + n], k, v, seen)
            assert_near(out[a:a + n], o, mass, f"request {r}")
            assert (out[a:a + n][~seen.any(-1)] == 0).all()
            a += n


LENS, KINDS = [700, 130, 300, 1000, 90, 5], ["some", "all", "none", "tail", "first", "all"]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 64, 128, 512])
@pytest.mark.parametrize("new,said", [(1, 1), (3, 3), (1, 1000), (3, 1000), (60, 1), (60, 60)])
@pytest.mark.parametrize("shared", [True, False])
def test_positions_without_a_page_are_not_seen(D, page, new, said, shared, workspace):
    """Whatever the launches before left on the chip: other requests' values, and numbers that are not finite."""
    c = Case(1, LENS, [min(new, n) for n in LENS], KINDS, 8, 2, D, page)
    ws = workspace if shared else None
    table, outs = c.table, []
    for fill in (math.nan, 3.0e4, -math.inf):
        c.table = c.full_table()
        c.run(said, ws, cache=torch.full_like(c.cache, fill))
        c.table = table
        outs.append(c.run(said, ws))
    check_errors()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    c.check(outs[0])


@pytest.mark.parametrize("new,said", [(1, 1), (5, 5), (5, 1000), (60, 60)])
def test_all_positions_that_have_a_page_seen(new, said, workspace):
    c = Case(2, LENS, [min(new, n) for n in LENS], KINDS, 8, 2, 128, 16)
    c.run(said, workspace, cache=torch.full_like(c.cache, math.nan))
    out = c.run(said, workspace, flags=mb.ATTENTION_FULL)
    check_errors()
    c.check(out, causal=False)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("new,said", [(3, 3), (3, 1000), (60, 60)])
def test_values_beside_positions_without_a_page(new, said, bad, workspace):
    """A value that is not finite still reaches exactly the tokens that see it."""
    c = Case(3, [316], [new], ["some"], 8, 2, 128, 8)
    clean = c.run(said, workspace)
    p = 316 - 2
    assert bool(c.there[0][p])
    c.cache[1][c.table[0, p // 8].long(), 1, p % 8, 10:20] = bad
    got = c.run(said, workspace)
    check_errors()
    assert torch.equal(got[:new - 2], clean[:new - 2]) and torch.equal(got[:, :4], clean[:, :4])
    hit = got[new - 2:, 4:, 10:20].float()
    assert (torch.isnan(hit) if bad != bad else hit == bad).all()


@pytest.mark.parametrize("D", [64, 128])
def test_a_pool_that_runs_out(D, workspace):
    """page_slots hands out what there is; the step's attention is over the positions that got a page."""
    page, H, G, new = 16, 4, 1, [40, 100, 1, 33]
    held = [0, 0, 0, 0]
    table = torch.full((4, 9), -1, dtype=torch.int32, device=DEV)
    pool = i32([3, 0, 5, 1, 6])  # 3 pages for the first request, 2 of 7 for the second, none after
    slots, positions, cu, lens, taken = mb.page_slots(i32(held), i32(new), table, pool, i32([0]), page, sum(new))
    assert int(taken) > pool.numel()
    g = torch.Generator(device=DEV).manual_seed(5)
    qkv = torch.randn(sum(new), (H + 2 * G) * D, generator=g, device=DEV)
    cache = torch.full((2, 8, G, page, D), math.nan, dtype=torch.bfloat16, device=DEV)
    turns, axes = mb.rope_turns(D, theta=1e4, device=DEV)
    q = mb.rope_kv(qkv, turns, positions, slots, cache[0], cache[1], H, axes=axes)
    for said in (100, 1):
        out = mb.attention_paged(q, cache[0], cache[1], table, lens, cu, said, workspace=workspace)
        check_errors()
        a = 0
        for r, n in enumerate(new):
            s = slots[a:a + n].long()
            there = s >= 0
            s = torch.where(there, s, 3 * page)
            k, v = (c[s // page, :, s % page] for c in cache)
            seen = there[None] & (torch.arange(n, device=DEV)[None] <= torch.arange(n, device=DEV)[:, None])
            assert_near(out[a:a + n], *formula(q[a:a + n], k, v, seen), f"request {r}, max_new {said}")
            a += n
        assert (out[140:] == 0).all()
