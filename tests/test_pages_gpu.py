"""Slots of a step's tokens and the way of the QKV heads into the cache, against plain implementations."""
import math

import pytest
import torch

import miori_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def check_errors():
    torch.cuda.synchronize()
    assert mb.lib.miori_device_error_poll() == 0


# ---- page_slots -----------------------------------------------------------------------------

def plain_slots(held, new, table, pool, taken, page, T):
    """Request by request, token by token."""
    table = [list(row) for row in table]
    width, given = len(table[0]), taken
    slots, positions, cu = [], [], [0]
    for r, (h, n) in enumerate(zip(held, new)):
        for i in range(min(-(-h // page), width), min(-(-(h + n) // page), width)):
            table[r][i] = pool[given] if given < len(pool) else -1
            given += 1
        for p in range(h, h + n):
            number = table[r][p // page] if p // page < width else -1
            slots.append(number * page + p % page if number >= 0 else -1)
            positions.append(p)
        cu.append(cu[-1] + n)
    pad = T - len(slots)
    return (slots + [-1] * pad)[:T], (positions + [0] * pad)[:T], cu, [h + n for h, n in zip(held, new)], given, table


def slots_case(held, new, page, width, pool_size, taken=0, spare=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(5000 + pool_size, generator=g).tolist()
    pool, rest = order[:pool_size], order[pool_size:]
    table, at = [], 0
    for h in held:
        own = min(-(-h // page), width)
        table.append((rest[at:at + own] + [-1] * width)[:width])
        at += own
    T = sum(new) + spare
    t = i32(table)
    before = [i32(held), i32(new), i32(pool), i32([taken])]
    got = mb.page_slots(before[0], before[1], t, before[2], before[3], page, T)
    check_errors()
    want = plain_slots(held, new, table, pool, taken, page, T)
    for name, a, b in zip(("slots", "positions", "cu", "held_after", "taken_after"), got, want):
        b = [b] if name == "taken_after" else b
        assert a.dtype == torch.int32 and a.tolist() == b, name
    assert t.tolist() == want[5]
    for x, y in zip(before, (held, new, pool, [taken])):
        assert x.tolist() == y


@pytest.mark.parametrize("page", [1, 3, 8, 16, 128])
def test_slots(page):
    slots_case([0, 15, 16, 17, 100, 0, 5], [1, 1, 1, 1, 40, 33, 0], page, 200, 300, taken=4, spare=6)
    slots_case([0], [1], page, 1, 1)
    slots_case([0, 0], [0, 0], page, 4, 1, spare=3)
    slots_case([3], [5000], page, 6000, 5500)


def test_many_requests():
    """More than the threads of a CTA, more tokens than one CTA takes, requests without tokens between them."""
    held = [(i * 37) % 90 for i in range(1300)]
    new = [(i * 7) % 5 for i in range(1300)]
    slots_case(held, new, 16, 8, 1500, spare=1)


def test_short_pools_tables_and_token_counts():
    slots_case([0, 0, 10], [40, 40, 40], 16, 10, 5)              # the pool ends inside the second request
    slots_case([0, 0, 10], [40, 40, 40], 16, 10, 5, taken=5)     # ... or is empty
    slots_case([30, 0], [40, 5], 16, 3, 50)                      # the table ends inside the first request
    slots_case([0, 9], [40, 5], 16, 5, 50, spare=-20)            # fewer rows than tokens


def test_slots_refusals():
    t = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    a, one = i32([1, 2]), i32([0])
    with pytest.raises(TypeError, match="int32"):
        mb.page_slots(a.long(), a, t, a, one, 16, 4)
    with pytest.raises(ValueError, match="numbers expected"):
        mb.page_slots(a, one, t, a, one, 16, 4)
    with pytest.raises(ValueError, match="table"):
        mb.page_slots(a, a, t[:1], a, one, 16, 4)
    with pytest.raises(mb.MioriError, match="empty table or page"):
        mb.page_slots(a, a, t, a, one, 0, 4)
    with pytest.raises(mb.MioriError, match="requests"):
        big = torch.zeros(16385, dtype=torch.int32, device=DEV)
        mb.page_slots(big, big, torch.zeros(16385, 1, dtype=torch.int32, device=DEV), a, one, 16, 4)


# ---- rope_kv ----------------------------------------------------------------------------------
# Tolerance, before the first run: the result is rounded to bf16 once (2^-8 of its value); what comes before is fp32.  A normed
# value is off by at most 2^-20 of itself (a sum of 128 squares, a reciprocal root, two products), a sine or cosine by 2^-22, and
# by 2 pi 2^-32 for the angle; so a turned pair (a, b) is off by 2^-18 (|a| + |b|) at most.

def plain_rope(qkv, turns, axes, positions, H, G, D, gamma_q, gamma_k, eps, adjacent):
    """64 bits; the angles as exact fractions of a turn.  Returns the heads and |a| + |b| of the pair that each element is of."""
    T, half = qkv.shape[0], len(turns)
    x = qkv.double().cpu().view(T, H + 2 * G, D)
    angle = torch.tensor([[2 * math.pi * ((p * t) % 2 ** 64) / 2 ** 64 for p, t in zip((row[a] for a in axes), turns)]
                          for row in positions.T.tolist()], dtype=torch.float64)[:, None]
    out, size = x.clone(), x.abs()
    a = torch.arange(half) * (2 if adjacent else 1)
    b = a + (1 if adjacent else half)
    for h, gamma in [(slice(0, H), gamma_q), (slice(H, H + G), gamma_k)]:
        y = x[:, h]
        if gamma is not None:
            y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * gamma.double().cpu()
        o, s = y.clone(), y.abs()
        o[..., a], o[..., b] = y[..., a] * angle.cos() - y[..., b] * angle.sin(), y[..., b] * angle.cos() + y[..., a] * angle.sin()
        s[..., a] = s[..., b] = y[..., a].abs() + y[..., b].abs()
        out[:, h], size[:, h] = o, s
    return out, size


def rope_case(T, H, G, D, rotary=None, axes=1, fp32=True, norm=True, adjacent=False, page=16, furthest=40000, seed=1, nhd=False, flags=0, pad=0):
    rotary = rotary or D
    g = torch.Generator(device=DEV).manual_seed(seed)
    wide = torch.randn(T, (H + 2 * G) * D + pad, generator=g, device=DEV).to(torch.float32 if fp32 else torch.bfloat16)
    qkv = wide[:, pad:]
    half = rotary // 2
    parts = [half // axes + (1 if a < half % axes else 0) for a in range(axes)]
    turns, ax = mb.rope_turns(rotary, theta=1e4, sections=parts, interleaved=axes == 3, device=DEV)
    positions = torch.randint(0, furthest, (axes, T), generator=g, device=DEV).to(torch.int32)
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:T].to(torch.int32)
    if T > 3:
        slots[1], slots[2] = -1, pages * page  # not kept
    cache = torch.randn(*((2, pages, page, G, D) if nhd else (2, pages, G, page, D)), generator=g, device=DEV).to(torch.bfloat16)
    cache = cache.transpose(2, 3) if nhd else cache
    was = cache.clone()
    gq, gk = ((torch.rand(2, D, generator=g, device=DEV) + 0.5).to(torch.bfloat16) if norm else (None, None))
    q = mb.rope_kv(qkv, turns, positions if axes > 1 else positions[0], slots, cache[0], cache[1], H, axes=ax, gamma_q=gq, gamma_k=gk, eps=1e-5,
                   flags=flags | (mb.ROPE_ADJACENT if adjacent else 0))
    check_errors()
    out, size = plain_rope(qkv, [t % 2 ** 64 for t in turns.tolist()], ax.tolist(), positions, H, G, D, gq, gk, 1e-5, adjacent)
    want = was.double().cpu()
    tol = torch.zeros_like(want)
    for i, h in ((0, slice(H, H + G)), (1, slice(H + G, H + 2 * G))):
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                want[i, s // page, :, s % page], tol[i, s // page, :, s % page] = out[t, h], size[t, h] * 2.0 ** -18 + out[t, h].abs() * 2.0 ** -8
    assert ((q.double().cpu() - out[:, :H]).abs() <= size[:, :H] * 2.0 ** -18 + out[:, :H].abs() * 2.0 ** -8).all(), "q"
    assert ((cache.double().cpu() - want).abs() <= tol).all(), "cache"
    return q, cache


@pytest.mark.parametrize("T", [1, 5, 77])
@pytest.mark.parametrize("H,G,D,rotary", [(16, 4, 128, 128), (16, 4, 128, 64), (3, 1, 64, 64), (8, 8, 64, 32), (5, 5, 128, 16), (1, 1, 64, 48)])
@pytest.mark.parametrize("fp32", [True, False])
def test_rope(T, H, G, D, rotary, fp32):
    rope_case(T, H, G, D, rotary, fp32=fp32)
    rope_case(T, H, G, D, rotary, axes=3, fp32=fp32, norm=False, adjacent=True, page=8, seed=2)


def test_rope_far_positions_and_other_layouts():
    rope_case(40, 4, 2, 128, axes=2, furthest=2 ** 31 - 1)
    rope_case(40, 4, 2, 64, axes=4, nhd=True, pad=64)
    rope_case(3000, 2, 1, 64)
    rope_case(9, 4, 2, 128, flags=mb.LAUNCH_PDL)


def test_rope_negative_positions_turn_back():
    turns, ax = mb.rope_turns(64, theta=1e4, device=DEV)
    x = torch.randn(2, 3 * 64, device=DEV)
    x[1] = x[0]
    cache = torch.zeros(2, 1, 1, 8, 64, dtype=torch.bfloat16, device=DEV)
    q = mb.rope_kv(x, turns, i32([5, -5]), i32([0, 1]), cache[0], cache[1], 1, axes=ax)
    a = x[0, :64].double().cpu()
    angle = torch.tensor([5.0 * 1e4 ** (-j / 32) for j in range(32)], dtype=torch.float64)
    want = torch.cat((a[:32] * angle.cos() + a[32:] * angle.sin(), a[32:] * angle.cos() - a[:32] * angle.sin()))
    size = (a[:32].abs() + a[32:].abs()).repeat(2)
    assert ((q[1, 0].double().cpu() - want).abs() <= size * 2.0 ** -18 + want.abs() * 2.0 ** -8).all()


def test_rope_leaves_the_rest_of_the_cache_alone_and_keeps_infinities():
    turns, ax = mb.rope_turns(64, theta=1e4, device=DEV)
    qkv = torch.randn(2, 3 * 64, device=DEV)
    qkv[0, 128:130] = torch.tensor([math.inf, math.nan])
    qkv[1, 3] = math.inf  # in q: its head is not finite, the other token's is
    cache = torch.full((2, 2, 1, 8, 64), 9.0, dtype=torch.bfloat16, device=DEV)
    q = mb.rope_kv(qkv, turns, i32([1, 2]), i32([3, 12]), cache[0], cache[1], 1, axes=ax)
    assert torch.isfinite(q[0].float()).all() and not torch.isfinite(q[1].float()).all()
    assert cache[1, 0, 0, 3, 0] == math.inf and torch.isnan(cache[1, 0, 0, 3, 1])
    cache[:, 0, 0, 3], cache[:, 1, 0, 4] = 9.0, 9.0
    assert (cache == 9.0).all()


def test_rope_refusals():
    turns, ax = mb.rope_turns(64, theta=1e4, device=DEV)
    x = torch.zeros(2, 4 * 64, device=DEV)
    cache = torch.zeros(2, 1, 1, 8, 64, dtype=torch.bfloat16, device=DEV)
    pos = i32([0, 1])
    with pytest.raises(ValueError, match="256 columns"):
        mb.rope_kv(x[:, :192], turns, pos, pos, cache[0], cache[1], 2)
    with pytest.raises(TypeError, match="fp32 or bf16"):
        mb.rope_kv(x.half(), turns, pos, pos, cache[0], cache[1], 2)
    with pytest.raises(TypeError, match="int64"):
        mb.rope_kv(x, turns.int(), pos, pos, cache[0], cache[1], 2)
    with pytest.raises(ValueError, match="positions"):
        mb.rope_kv(x, turns, pos[:1], pos, cache[0], cache[1], 2)
    with pytest.raises(ValueError, match="weights expected"):
        mb.rope_kv(x, turns, pos, pos, cache[0], cache[1], 2, gamma_q=torch.zeros(32, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="differ in shape"):
        mb.rope_kv(x, turns, pos, pos, cache[0], cache[1, :, :, :4], 2)
    with pytest.raises(mb.MioriError, match="rotary"):
        mb.rope_kv(x, torch.zeros(64, dtype=torch.int64, device=DEV), pos, pos, cache[0], cache[1], 2)
    with pytest.raises(mb.MioriError, match="four axes"):
        mb.rope_kv(x, turns, torch.zeros(5, 2, dtype=torch.int32, device=DEV), pos, cache[0], cache[1], 2)
    check_errors()
