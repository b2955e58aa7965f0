"""The attention of a decode step and of a prompt, with the page cache between them, as cases that can be timed and compared.

Sizes are those of the benchmark's model (QKV 2048 -> 3072: 16 query heads of 128 over 4 key heads; 32 slots; 1024 tokens
packed of 32 prompts; 64 prompts of 2048) and generic ones around them, odd and ragged ones included.  A kind is one operator:

  slots   `page_slots`        positions, cache slots and new pages of the tokens of a step, from the requests' lengths
  rope    `rope_kv`           QKV row -> heads normed and turned by their positions, keys and values into their cache slots
  paged   `attention_paged`   one new token per request (decoding) or a chunk of them over a paged cache
  prompt  `attention_prompt`  whole prompts, packed one behind the other, causal

Where `own` is false, `run` computes the plain form: elementary operations of torch over padded tensors, in 32 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
WORKSPACE = 64 << 20  # what a program that calls the attention operators keeps for them
EPS = 1e-5
THETA = 1e6
TURN = 2.0 * math.pi / 2.0 ** 64  # an angle as a whole number of these


def listed():
    return [
        # a decode step of all 32 slots, each with one new token
        {"name": "slots-decode", "kind": "slots", "requests": 32, "held": 3000, "new": 1, "lengths": 1, "page": 16, "spare": 0},
        # 64 new prompts of up to 2048 tokens, and one of them continued
        {"name": "slots-prompts", "kind": "slots", "requests": 64, "held": 0, "new": 2048, "lengths": 2, "page": 64, "spare": 77},
        # one decode step behind the QKV projection, whose outputs are fp32: normed heads, three axes (time, height, width)
        {"name": "rope-decode", "kind": "rope", "tokens": 32, "heads": 16, "kv_heads": 4, "dim": 128, "rotary": 128, "axes": 3,
         "norm": True, "fp32": True, "adjacent": False, "page": 16, "furthest": 32768},
        # a long prompt with images in it, from a projection that rounded to bf16
        {"name": "rope-prompt", "kind": "rope", "tokens": 16384, "heads": 16, "kv_heads": 4, "dim": 128, "rotary": 128, "axes": 3,
         "norm": True, "fp32": False, "adjacent": False, "page": 64, "furthest": 16384},
        # one stream in the middle of an answer: latency counts
        {"name": "decode-one", "kind": "paged", "requests": 1, "heads": 16, "kv_heads": 4, "dim": 128, "page": 16, "held": 1000, "new": 1,
         "lengths": 5},
        # all slots full, contexts of very different lengths: the cache's bytes count
        {"name": "decode-slots", "kind": "paged", "requests": 32, "heads": 16, "kv_heads": 4, "dim": 128, "page": 16, "held": 32768, "new": 1,
         "lengths": 6},
        # a few drafted tokens per request, checked together; narrow heads
        {"name": "draft-check", "kind": "paged", "requests": 9, "heads": 32, "kv_heads": 8, "dim": 64, "page": 32, "held": 5000, "new": 5,
         "lengths": 7},
        # chunks of long prompts beside short ones
        {"name": "chunk", "kind": "paged", "requests": 4, "heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "held": 16384, "new": 512,
         "lengths": 8},
        # one short prompt
        {"name": "prompt-77", "kind": "prompt", "prompts": 1, "heads": 16, "kv_heads": 4, "dim": 128, "tokens": 77, "ragged": False, "lengths": 9},
        # 32 prompts of 32 tokens packed
        {"name": "prompts-packed", "kind": "prompt", "prompts": 32, "heads": 16, "kv_heads": 4, "dim": 128, "tokens": 32, "ragged": False,
         "lengths": 10},
        # ordinary prompts, narrow heads
        {"name": "prompts-narrow", "kind": "prompt", "prompts": 8, "heads": 32, "kv_heads": 8, "dim": 64, "tokens": 2048, "ragged": True,
         "lengths": 11},
        # documents
        {"name": "prompts-long", "kind": "prompt", "prompts": 4, "heads": 16, "kv_heads": 4, "dim": 128, "tokens": 8192, "ragged": True,
         "lengths": 12},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))

    kind = rng.choice(("slots", "rope", "paged", "prompt"))
    lengths = rng.randrange(1 << 20)
    if kind == "slots":
        return {"kind": kind, "requests": spread(1, 256), "held": rng.choice((0, spread(1, 30000))), "new": spread(1, 2048), "lengths": lengths,
                "page": rng.choice((8, 16, 32, 64, 128)), "spare": rng.choice((0, spread(1, 500)))}
    heads, kv_heads, dim = rng.choice(((16, 4, 128), (32, 8, 64), (16, 16, 64), (12, 2, 128), (20, 4, 64), (16, 1, 128), (15, 5, 128), (8, 8, 128), (28, 4, 128)))
    if kind == "rope":
        return {"kind": kind, "tokens": spread(1, 16384), "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice((dim, dim // 2)),
                "axes": rng.choice((1, 2, 3)), "norm": rng.random() < 0.7, "fp32": rng.random() < 0.5, "adjacent": rng.random() < 0.3,
                "page": rng.choice((8, 16, 32, 64, 128)), "furthest": spread(100, 200000)}
    if kind == "paged":
        requests = spread(1, 48)
        most = 32 * 32768 // requests  # positions that the plain form pads its requests to
        held = spread(16, min(65536, most))
        new = rng.choice((1, 1, spread(2, 16), spread(2, 600)))
        new = max(1, min(new, 512 * 4 * 16384 // (requests * (held + 600))))
        return {"kind": kind, "requests": requests, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice((8, 16, 32, 64, 128)),
                "held": held, "new": new, "lengths": lengths}
    prompts = spread(1, 64)
    most = int(math.sqrt(4 * 8192 * 8192 * 16 / (prompts * heads)))
    return {"kind": kind, "prompts": prompts, "heads": heads, "kv_heads": kv_heads, "dim": dim, "tokens": spread(1, min(8192, most)),
            "ragged": rng.random() < 0.7, "lengths": lengths}


# ---- lengths: a case's own, the same for every seed ------------------------------------

def _ragged(count, most, key, least=1):
    """Lengths from `least` to `most`, spread over their logarithm for half of them; the longest is `most`."""
    rng = random.Random(key)
    got = [most if i == 0 else int(rng.uniform(least, most)) if rng.random() < 0.5 else int(round(math.exp(rng.uniform(math.log(max(least, 1)), math.log(max(most, 1))))))
           for i in range(count)]
    rng.shuffle(got)
    return [max(least, min(most, n)) for n in got]


def _request_lengths(c):
    """(held, new) of a case's requests."""
    n = c["requests"]
    held = _ragged(n, c["held"], c["lengths"], 0) if c["held"] else [0] * n
    new = [1] * n if c["new"] == 1 else _ragged(n, c["new"], c["lengths"] + 1)
    return held, new


def _prompt_lengths(c):
    return _ragged(c["prompts"], c["tokens"], c["lengths"]) if c["ragged"] else [c["tokens"]] * c["prompts"]


def _pages(n, page):
    return -(-n // page)


# ---- what a program has in hand ----------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cu(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return _ints(cu)


def _heads(g, tokens, heads, dim):
    """Normed heads: unit variance with a spread of scales over the dimensions, as behind a head norm."""
    scale = torch.rand(heads, dim, generator=g, device=DEV) + 0.5
    return (torch.randn(tokens, heads, dim, generator=g, device=DEV) * scale).to(torch.bfloat16)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    if c["kind"] == "slots":
        held, new = _request_lengths(c)
        page = c["page"]
        owned = [_pages(n, page) for n in held]
        width = max(_pages(a + b, page) for a, b in zip(held, new)) + 3
        total = sum(_pages(a + b, page) for a, b in zip(held, new)) + 50
        pages = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        table = torch.full((c["requests"], width), -1, dtype=torch.int32, device=DEV)
        rows = torch.tensor([r for r, n in enumerate(owned) for _ in range(n)], dtype=torch.long, device=DEV)
        cols = torch.tensor([i for n in owned for i in range(n)], dtype=torch.long, device=DEV)
        table[rows, cols] = pages[:sum(owned)]
        taken = 7  # some of the free list is given away already
        pool = torch.cat((pages[:taken], pages[sum(owned):]))
        return {"c": c, "held": _ints(held), "new": _ints(new), "table": table, "pool": pool.contiguous(), "taken": _ints([taken]),
                "T": sum(new) + c["spare"]}
    if c["kind"] == "rope":
        T, H, G, D = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        qkv = torch.randn(T, (H + 2 * G) * D, generator=g, device=DEV) * (torch.rand((H + 2 * G) * D, generator=g, device=DEV) + 0.5)
        qkv = qkv if c["fp32"] else qkv.to(torch.bfloat16)
        half = c["rotary"] // 2
        turns = torch.tensor([int(THETA ** (-j / half) / TURN) for j in range(half)], dtype=torch.long, device=DEV)
        # the axes share the frequencies: a block of them each, the first takes what is left
        part = half // c["axes"]
        axes = _ints([max(0, c["axes"] - 1 - (half - 1 - j) // part) for j in range(half)])
        # runs of text, where all axes count together, and of image, where height and width walk a grid of 24 columns
        first = torch.randint(0, c["furthest"] - min(T, c["furthest"] - 1), (1,), generator=g, device=DEV)
        t = torch.arange(T, device=DEV)
        image = (t // 96) % 2 == 1
        i = t % 96
        pos = torch.stack([first + t, torch.where(image, first + t - i + i // 24, first + t), torch.where(image, first + t - i + i % 24, first + t)])
        pos[0] = torch.where(image, first + t - i, first + t)
        pages = _pages(T, c["page"]) + 3
        where = torch.randperm(pages, generator=g, device=DEV)
        slots = where[t // c["page"]] * c["page"] + t % c["page"]
        cache = torch.randn(2, pages, G, c["page"], D, generator=g, device=DEV).to(torch.bfloat16)
        gamma = (1 + 0.2 * torch.randn(2, D, generator=g, device=DEV)).to(torch.bfloat16)
        return {"c": c, "qkv": qkv, "turns": turns, "axes": axes, "positions": pos[:c["axes"]].to(torch.int32).contiguous(), "slots": slots.to(torch.int32),
                "k_cache": cache[0], "v_cache": cache[1], "gamma_q": gamma[0] if c["norm"] else None, "gamma_k": gamma[1] if c["norm"] else None}
    if c["kind"] == "paged":
        held, new = _request_lengths(c)
        H, G, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
        owned = [_pages(a + b, page) for a, b in zip(held, new)]
        total = sum(owned) + 5
        pages = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        table = torch.zeros((c["requests"], max(owned)), dtype=torch.int32, device=DEV)
        rows = torch.tensor([r for r, n in enumerate(owned) for _ in range(n)], dtype=torch.long, device=DEV)
        cols = torch.tensor([i for n in owned for i in range(n)], dtype=torch.long, device=DEV)
        table[rows, cols] = pages[:sum(owned)]
        cache = torch.empty(2, total, G, page, D, dtype=torch.bfloat16, device=DEV)
        for half in cache:
            half.normal_(generator=g)
        return {"c": c, "q": _heads(g, sum(new), H, D), "k_cache": cache[0], "v_cache": cache[1], "table": table,
                "lens": _ints([a + b for a, b in zip(held, new)]), "cu": _cu(new), "max_new": max(new),
                "workspace": torch.zeros(WORKSPACE, dtype=torch.uint8, device=DEV)}
    lengths = _prompt_lengths(c)
    T = sum(lengths)
    return {"c": c, "q": _heads(g, T, c["heads"], c["dim"]), "k": _heads(g, T, c["kv_heads"], c["dim"]),
            "v": torch.randn(T, c["kv_heads"], c["dim"], generator=g, device=DEV).to(torch.bfloat16), "cu": _cu(lengths), "longest": max(lengths),
            "workspace": torch.zeros(WORKSPACE, dtype=torch.uint8, device=DEV)}


# ---- the framework's calls -----------------------------------------------------------------

def _own_pass(s):
    import miori_b200 as mb
    c = s["c"]
    if c["kind"] == "slots":
        return (*mb.page_slots(s["held"], s["new"], s["table"], s["pool"], s["taken"], c["page"], s["T"]), s["table"])
    if c["kind"] == "rope":
        q = mb.rope_kv(s["qkv"], s["turns"], s["positions"], s["slots"], s["k_cache"], s["v_cache"], c["heads"], axes=s["axes"],
                       gamma_q=s["gamma_q"], gamma_k=s["gamma_k"], eps=EPS, flags=mb.ROPE_ADJACENT if c["adjacent"] else 0)
        return q, s["k_cache"], s["v_cache"]
    if c["kind"] == "paged":
        return mb.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"], s["max_new"], workspace=s["workspace"])
    return mb.attention_prompt(s["q"], s["k"], s["v"], s["cu"], workspace=s["workspace"])


# ---- the plain forms ------------------------------------------------------------------------

def _request_of(cu, T):
    """(request, index in it) of each of T packed tokens; those past the end count to the last request."""
    t = torch.arange(T, device=DEV)
    r = (t[:, None] >= cu[1:-1]).sum(1)
    return r, t - cu[r]


def _plain_slots(held, new, table, pool, taken, page, T):
    cu = torch.cat((torch.zeros_like(taken), torch.cumsum(new, 0, dtype=torch.int32)))
    after = held + new
    own_before, own_after = (held + page - 1) // page, (after + page - 1) // page
    wanted = own_after - own_before
    first = taken + torch.cumsum(wanted, 0, dtype=torch.int32) - wanted
    col = torch.arange(table.shape[1], device=DEV)
    fresh = (col >= own_before[:, None]) & (col < own_after[:, None])
    given = pool[(first[:, None] + col - own_before[:, None]).clamp(0, pool.numel() - 1)]
    table.copy_(torch.where(fresh, given, table))
    r, i = _request_of(cu, T)
    position = held[r] + i
    slot = table[r, (position // page).clamp(max=table.shape[1] - 1)] * page + position % page
    there = torch.arange(T, device=DEV) < cu[-1]
    return (torch.where(there, slot, -1).to(torch.int32), torch.where(there, position, 0).to(torch.int32), cu, after, taken + wanted.sum(dtype=torch.int32), table)


def _plain_rope(s, c):
    T, H, G, D, R = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rotary"]
    x = s["qkv"].float().view(T, H + 2 * G, D)
    qk, v = x[:, :H + G], x[:, H + G:]
    if s["gamma_q"] is not None:
        gamma = torch.cat((s["gamma_q"].float().expand(H, D), s["gamma_k"].float().expand(G, D)))
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * gamma
    phase = s["positions"].long()[s["axes"].long()].T * s["turns"]  # whole turns fall off
    angle = phase.float() * TURN
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    if c["adjacent"]:
        a, b = qk[..., 0:R:2], qk[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = qk[..., :R // 2], qk[..., R // 2:R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    qk = torch.cat((turned, qk[..., R:]), -1).to(torch.bfloat16)
    page, at = s["slots"].long() // c["page"], s["slots"].long() % c["page"]
    s["k_cache"][page, :, at] = qk[:, H:]
    s["v_cache"][page, :, at] = v.to(torch.bfloat16)
    return qk[:, :H].contiguous(), s["k_cache"], s["v_cache"]


def _plain_attention(q, k, v, count, lens):
    """q [B][n][H][D], k and v [B][L][G][D], fp32; request b has count[b] queries, the last of its lens[b] positions."""
    B, n, H, D = q.shape
    L, G = k.shape[1:3]
    scores = torch.matmul(q.view(B, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * n, D), k.permute(0, 2, 3, 1)).view(B, G, H // G, n, L)
    last = (lens - count)[:, None] + torch.arange(n, device=DEV)  # position of each query
    seen = torch.arange(L, device=DEV) <= last[:, :, None]
    scores = scores.mul_(1.0 / math.sqrt(D)).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, G, H // G * n, L), v.permute(0, 2, 1, 3)).view(B, G, H // G, n, D) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)


def _padded(x, cu, most):
    at = (cu[:-1, None] + torch.arange(most, device=DEV)).clamp(max=x.shape[0] - 1)
    return x[at].float()


def _plain_pass(s):
    c = s["c"]
    if c["kind"] == "slots":
        return _plain_slots(s["held"], s["new"], s["table"], s["pool"], s["taken"], c["page"], s["T"])
    if c["kind"] == "rope":
        return _plain_rope(s, c)
    cu = s["cu"]
    count = cu[1:] - cu[:-1]
    if c["kind"] == "paged":
        R, W = s["table"].shape
        k, v = (x[s["table"]].permute(0, 1, 3, 2, 4).reshape(R, W * c["page"], c["kv_heads"], c["dim"]).float() for x in (s["k_cache"], s["v_cache"]))
        o = _plain_attention(_padded(s["q"], cu, s["max_new"]), k, v, count, s["lens"])
    else:
        o = _plain_attention(*(_padded(s[x], cu, s["longest"]) for x in "qkv"), count, count)
    return o[_request_of(cu, s["q"].shape[0])].to(torch.bfloat16)


def run(state):
    return _own_pass(state) if own else _plain_pass(state)


# ---- what a pass cannot do without -----------------------------------------------------------

def _seen(count, length):
    """Sum over the queries of a request of the positions that each sees."""
    return count * (length - count) + count * (count + 1) // 2


def work(case):
    c = case
    if c["kind"] == "slots":
        held, new = _request_lengths(c)
        pages = sum(_pages(a + b, c["page"]) - _pages(a, c["page"]) for a, b in zip(held, new))
        partial = sum(1 for a in held if a % c["page"])  # pages that are there already and take a token
        return {"bytes": 4 * (2 * c["requests"] + pages + partial + 1) + 4 * (pages + 2 * c["requests"] + 2) + 8 * (sum(new) + c["spare"]),
                "flops": 2 * (sum(new) + c["spare"]) + 8 * c["requests"]}
    if c["kind"] == "rope":
        T, H, G, D = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        values = T * (H + 2 * G) * D
        small = 4 * T * (c["axes"] + 1) + 6 * c["rotary"] + (4 * D if c["norm"] else 0)
        return {"bytes": values * ((4 if c["fp32"] else 2) + 2) + small, "flops": T * (H + G) * (3 * c["rotary"] + (4 * D if c["norm"] else 0))}
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "paged":
        held, new = _request_lengths(c)
        kv = 4 * G * D * sum(a + b for a, b in zip(held, new))
        pairs = sum(_seen(b, a + b) for a, b in zip(held, new))
        table = 4 * sum(_pages(a + b, c["page"]) for a, b in zip(held, new)) + 8 * c["requests"]
        return {"bytes": kv + 4 * H * D * sum(new) + table, "flops": 4 * H * D * pairs}
    lengths = _prompt_lengths(c)
    return {"bytes": 4 * (H + G) * D * sum(lengths) + 4 * len(lengths), "flops": 4 * H * D * sum(_seen(n, n) for n in lengths)}


# ---- 64 bits, request by request -----------------------------------------------------------

def _exact_attention(q, k, v, first):
    """One request: q [n][H][D] at positions first, first + 1, ...; k and v [L][G][D].  A block of queries at a time."""
    n, H, D = q.shape
    G = k.shape[1]
    out = torch.empty(n, H, D, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 28) // max(1, k.shape[0] * (H // G)))
    for h in range(G):
        kh, vh = k[:, h].double(), v[:, h].double()
        for a in range(0, n, step):
            b = min(n, a + step)
            end = first + b  # the last of these sees so many positions
            x = torch.einsum("nhd,ld->nhl", q[a:b, h * (H // G):(h + 1) * (H // G)].double(), kh[:end]) / D ** 0.5
            hidden = torch.arange(end, device=DEV)[None, :] > first + torch.arange(a, b, device=DEV)[:, None]
            w = torch.softmax(x.masked_fill(hidden[:, None], -math.inf), -1)
            out[a:b, h * (H // G):(h + 1) * (H // G)] = torch.einsum("nhl,ld->nhd", w, vh[:end])
    return out


def exact(case, seed):
    c = case
    if c["kind"] == "slots":
        return None  # whole numbers
    s = prepare(case, seed)
    if c["kind"] == "rope":
        T, H, G, D, R = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rotary"]
        half = R // 2
        x = s["qkv"].double().reshape(T, H + 2 * G, D)
        # the angle's fraction of a turn: the upper and lower halves of the 64-bit step, each exact in a double for positions below 2^21
        p = s["positions"].double()[s["axes"].long()].T
        upper, lower = (s["turns"] >> 32).double(), (s["turns"] & 0xFFFFFFFF).double()
        angle = 2 * math.pi * (torch.remainder(p * upper / 2.0 ** 32, 1.0) + p * lower / 2.0 ** 64)[:, None]
        first = torch.arange(half, device=DEV) * (2 if c["adjacent"] else 1)
        second = first + (1 if c["adjacent"] else half)
        heads = []
        for part, gamma in ((x[:, :H], s["gamma_q"]), (x[:, H:H + G], s["gamma_k"])):
            if gamma is not None:
                part = part / torch.sqrt((part ** 2).sum(-1, keepdim=True) / D + EPS) * gamma.double()
            turned = part.clone()
            turned[..., first] = part[..., first] * angle.cos() - part[..., second] * angle.sin()
            turned[..., second] = part[..., first] * angle.sin() + part[..., second] * angle.cos()
            heads.append(turned)
        caches = []
        for cache, rows in ((s["k_cache"], heads[1]), (s["v_cache"], x[:, H + G:])):
            whole = cache.double()
            whole[s["slots"].long() // c["page"], :, s["slots"].long() % c["page"]] = rows
            caches.append(whole)
        return (heads[0], *caches)
    if c["kind"] == "paged":
        held, new = _request_lengths(c)
        done, parts = 0, []
        for r, (a, b) in enumerate(zip(held, new)):
            pages = s["table"][r, :_pages(a + b, c["page"])].long()
            k, v = (x[pages].transpose(1, 2).reshape(-1, c["kv_heads"], c["dim"])[:a + b] for x in (s["k_cache"], s["v_cache"]))
            parts.append(_exact_attention(s["q"][done:done + b], k, v, a))
            done += b
        return torch.cat(parts)
    done, parts = 0, []
    for n in _prompt_lengths(c):
        parts.append(_exact_attention(*(s[x][done:done + n] for x in "qkv"), 0))
        done += n
    return torch.cat(parts)
