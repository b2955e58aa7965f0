"""Products in 8-bit floating point and layers of experts, as cases that can be timed and compared.

Sizes are those of the benchmark's model (hidden 2048, feed-forward 8192, gate + up 16384; 32 slots; prompts of 77
and of a thousand tokens, 16384 packed) and generic ones around them, odd and ragged ones included.  A kind is one operator:

  quant  `quant_fp8`         rows, or tiles of 128 rows, as 8-bit floating point with a scale for each block of 128
  gemm   `gemm_fp8`          rows in such blocks times weights in tiles of 128 x 128, one row (decoding) to packed prompts
  moe    `moe4`, `moe_fp8`   a whole layer of experts for the tokens of a decode step: router, choice, experts, weighted sum;
                             weights packed in 4 bits or in 8-bit floating point

Where `own` is false, `run` computes the plain form: elementary operations of torch, in 32 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
WORKSPACE = 64 << 20  # what a program that calls the layers of experts keeps for them
BLOCK = 128
TOP = 448.0  # the largest finite value of the type
LEAST = 2.0 ** -100  # a block's largest magnitude counts as no less
FP8 = torch.float8_e4m3fn
LARGEST_GEMM = 16384 * 16384 * 2048
LARGEST_EXPERTS = 32 * 2048 * 1536


def listed():
    return [
        # the activations of 32 slots in front of a projection: latency counts
        {"name": "quant-slots", "kind": "quant", "rows": 32, "K": 2048, "tile": 1, "fp32": False},
        # packed prompts in front of the feed-forward's second projection
        {"name": "quant-prompts", "kind": "quant", "rows": 16384, "K": 8192, "tile": 1, "fp32": False},
        # start-up: the widest weights of a layer, from what `dequant4_rowmajor` gives
        {"name": "quant-weights", "kind": "quant", "rows": 16384, "K": 2048, "tile": 128, "fp32": False},
        # decoding of one stream: the smallest product
        {"name": "gemm-1row", "kind": "gemm", "M": 1, "N": 2048, "K": 2048, "bf16": False},
        # eight slots and the widest weights: their bytes count
        {"name": "gemm-8rows", "kind": "gemm", "M": 8, "N": 16384, "K": 2048, "bf16": True},
        # one short prompt; a K that ends inside a block, an N that is no multiple of anything
        {"name": "gemm-ragged", "kind": "gemm", "M": 77, "N": 5003, "K": 1440, "bf16": False},
        # a thousand tokens packed, long rows
        {"name": "gemm-1024tokens", "kind": "gemm", "M": 1024, "N": 2048, "K": 8192, "bf16": True},
        # large packed prompts, the widest weights: the matrix units' rate counts
        {"name": "gemm-16384tokens", "kind": "gemm", "M": 16384, "N": 16384, "K": 2048, "bf16": True},
        # one stream through 4 of 32 packed experts, chosen by sigmoids with a bias
        {"name": "moe4-1token", "kind": "moe", "bits": 4, "group": 64, "tokens": 1, "experts": 32, "top": 4, "hidden": 2048, "ff": 1536, "sigmoid": True,
         "bias": True, "norm": True},
        # all slots: nearly every expert is some token's
        {"name": "moe4-32tokens", "kind": "moe", "bits": 4, "group": 64, "tokens": 32, "experts": 32, "top": 4, "hidden": 2048, "ff": 1536, "sigmoid": True,
         "bias": True, "norm": True},
        # a few streams, many narrow experts in 8-bit floating point, chosen by a softmax
        {"name": "moe8-4tokens", "kind": "moe", "bits": 8, "group": 128, "tokens": 4, "experts": 64, "top": 8, "hidden": 2048, "ff": 768, "sigmoid": False,
         "bias": False, "norm": True},
        # odd numbers of tokens and experts, rows that end inside a block
        {"name": "moe8-ragged", "kind": "moe", "bits": 8, "group": 128, "tokens": 13, "experts": 20, "top": 3, "hidden": 1440, "ff": 720, "sigmoid": False,
         "bias": True, "norm": False},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))

    kind = rng.choice(("quant", "gemm", "moe"))
    if kind == "quant":
        K = spread(64, 16384)
        return {"kind": kind, "rows": spread(1, min(16384, (1 << 27) // K)), "K": K, "tile": rng.choice((1, 1, 128)), "fp32": rng.random() < 0.3}
    if kind == "gemm":
        N, K = spread(64, 16384), 16 * spread(4, 512)
        M = rng.choice((spread(1, 64), spread(1, 16384)))
        return {"kind": kind, "M": max(1, min(M, LARGEST_GEMM // (N * K))), "N": N, "K": K, "bf16": rng.random() < 0.5}
    bits = rng.choice((4, 4, 8))
    step = 128 if bits == 4 else 16  # what rows are multiples of
    hidden = step * max(1, spread(512, 4096) // step)
    ff = step * max(1, spread(256, 2560) // step)
    experts = max(1, min(rng.choice((8, 16, 20, 32, 64, 128)), LARGEST_EXPERTS // (hidden * ff)))
    return {"kind": kind, "bits": bits, "group": rng.choice((32, 64)) if bits == 4 else 128, "tokens": spread(1, 32), "experts": experts,
            "top": min(experts, rng.choice((1, 2, 3, 4, 6, 8))), "hidden": hidden, "ff": ff, "sigmoid": rng.random() < 0.5, "bias": rng.random() < 0.5,
            "norm": rng.random() < 0.6}


def _blocks(n):
    return -(-n // BLOCK)


# ---- what a program has in hand ----------------------------------------------------------

def _whole_blocks(x, tile):
    """[rows][K] as [row blocks][tile][column blocks][128], zeros behind the ends."""
    rows, K = x.shape
    R = -(-rows // tile)
    x = torch.nn.functional.pad(x, (0, _blocks(K) * BLOCK - K, 0, R * tile - rows))
    return x.view(R, tile, _blocks(K), BLOCK)


def _quantized(x, tile):
    """(values, scales) of the blocks of x, tile x 128 elements each; rows of the values begin on 16-byte boundaries."""
    blocks = _whole_blocks(x.float(), tile)
    top = blocks.abs().amax((1, 3)).clamp(min=LEAST)
    most = torch.full_like(top, TOP)  # a plain number would be divided by as a product with its reciprocal
    q = (blocks * (most / top)[:, None, :, None]).to(FP8).flatten(2).flatten(0, 1)
    return q[:x.shape[0], :x.shape[1]], top / most


def _activations(g, rows, K):
    """Normed rows: unit variance, a spread of scales over the columns, some rows larger than others."""
    return torch.randn(rows, K, generator=g, device=DEV) * (torch.rand(K, generator=g, device=DEV) + 0.5) * (0.25 + 2 * torch.rand(rows, 1, generator=g, device=DEV))


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    if c["kind"] == "quant":
        x = _activations(g, c["rows"], c["K"])
        return {"c": c, "x": x if c["fp32"] else x.to(torch.bfloat16)}
    if c["kind"] == "gemm":
        a, sa = _quantized(_activations(g, c["M"], c["K"]), 1)
        w, sw = _quantized(torch.randn(c["N"], c["K"], generator=g, device=DEV) * 0.02, BLOCK)
        return {"c": c, "a": a, "sa": sa, "w": w, "sw": sw}
    T, E, H, F = c["tokens"], c["experts"], c["hidden"], c["ff"]
    s = {"c": c, "x": _activations(g, T, H).to(torch.bfloat16), "router": (torch.randn(E, H, generator=g, device=DEV) / H ** 0.5).to(torch.bfloat16),
         "bias": 0.1 * torch.randn(E, generator=g, device=DEV) if c["bias"] else None}
    for name, N, K in (("up", 2 * F, H), ("down", H, F)):
        if c["bits"] == 4:
            codes = torch.randint(-2 ** 31, 2 ** 31, (E, N, K // 8), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
            scale = (0.02 / 4.6 * (0.5 + torch.rand(E, N, K // c["group"], generator=g, device=DEV))).to(torch.bfloat16)
            least = (-7.5 * scale.float() * (0.9 + 0.2 * torch.rand(scale.shape, generator=g, device=DEV))).to(torch.bfloat16)
            s[name] = (codes, scale, least)
        else:
            w = torch.empty(E, N, K, dtype=FP8, device=DEV)
            w.copy_((torch.randn(E, N, K, generator=g, device=DEV) * 100).clamp_(-TOP, TOP))
            s[name] = (w, 0.02 / 100 * (0.5 + torch.rand(E, _blocks(N), _blocks(K), generator=g, device=DEV)))
    s["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device=DEV)
    return s


# ---- the framework's calls -----------------------------------------------------------------

def _own_pass(s):
    import miori_b200 as mb
    c = s["c"]
    if c["kind"] == "quant":
        return mb.quant_fp8(s["x"], tile=c["tile"])
    if c["kind"] == "gemm":
        return mb.gemm_fp8(s["a"], s["sa"], s["w"], s["sw"], flags=mb.OUT_BF16 if c["bf16"] else 0)
    flags = mb.OUT_BF16 | (mb.MOE_SIGMOID if c["sigmoid"] else 0) | (mb.MOE_NORM if c["norm"] else 0)
    if c["bits"] == 4:
        return mb.moe4(s["x"], s["router"], *s["up"], *s["down"], c["top"], s["workspace"], bias=s["bias"], group=c["group"], flags=flags)
    return mb.moe_fp8(s["x"], s["router"], *s["up"], *s["down"], c["top"], s["workspace"], bias=s["bias"], flags=flags)


# ---- the plain forms ------------------------------------------------------------------------

def _spread_tiles(scale, N, K, rows=BLOCK):
    """A block's scale at each of its elements: [..][N][K]."""
    return scale.repeat_interleave(rows, -2)[..., :N, :].repeat_interleave(BLOCK, -1)[..., :K]


def _weights(kept, c):
    """fp32 weights of some experts, [..][N][K]."""
    if c["bits"] == 8:
        w, scale = kept
        return w.float() * _spread_tiles(scale, *w.shape[-2:])
    words, scale, least = kept
    codes = (words[..., None] >> torch.arange(0, 32, 4, device=DEV, dtype=torch.int32)) & 15
    codes = codes.flatten(-2).unflatten(-1, (-1, c["group"])).float()
    return (codes * scale.float()[..., None] + least.float()[..., None]).flatten(-2)


def _choice(s, c):
    """(experts, weights) [tokens][top] of each token; the scores in 64 bits, since a choice hangs on them."""
    logits = s["x"].double() @ s["router"].double().T
    p = torch.sigmoid(logits) if c["sigmoid"] else torch.softmax(logits, -1)
    chosen = torch.topk(p if s["bias"] is None else p + s["bias"], c["top"], -1).indices
    w = p.gather(-1, chosen)
    return chosen, (w / w.sum(-1, keepdim=True) if c["norm"] else w).float()


def _plain_pass(s):
    c = s["c"]
    if c["kind"] == "quant":
        return _quantized(s["x"], c["tile"])
    if c["kind"] == "gemm":
        a, w = s["a"].float() * _spread_tiles(s["sa"], c["M"], c["K"], 1), s["w"].float() * _spread_tiles(s["sw"], c["N"], c["K"])
        return (a @ w.T).to(torch.bfloat16 if c["bf16"] else torch.float32)
    chosen, weight = _choice(s, c)
    T, F = c["tokens"], c["ff"]
    if T * c["top"] < c["experts"]:  # the chosen experts, one for each (token, place)
        e = chosen.flatten()
        x = s["x"].float().repeat_interleave(c["top"], 0)[:, None]
        up, down = (_weights([t[e] for t in s[name]], c) for name in ("up", "down"))
        gu = torch.matmul(x, up.transpose(-1, -2))
        y = torch.matmul(torch.nn.functional.silu(gu[..., :F]) * gu[..., F:], down.transpose(-1, -2)).view(T, c["top"], -1)
        return (y * weight[..., None]).sum(1).to(torch.bfloat16)
    share = torch.zeros(T, c["experts"], device=DEV).scatter_(1, chosen, weight)
    gu = torch.matmul(s["x"].float(), _weights(s["up"], c).transpose(-1, -2))
    y = torch.matmul(torch.nn.functional.silu(gu[..., :F]) * gu[..., F:], _weights(s["down"], c).transpose(-1, -2))
    return (y * share.T[..., None]).sum(0).to(torch.bfloat16)


def run(state):
    return _own_pass(state) if own else _plain_pass(state)


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "quant":
        n = c["rows"] * c["K"]
        return {"bytes": n * (5 if c["fp32"] else 3) + 4 * -(-c["rows"] // c["tile"]) * _blocks(c["K"]), "flops": 2 * n}
    if c["kind"] == "gemm":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": (M + N) * K + 4 * _blocks(K) * (M + _blocks(N)) + M * N * (2 if c["bf16"] else 4), "flops": 2 * M * N * K}
    T, E, H, F, top = c["tokens"], c["experts"], c["hidden"], c["ff"], c["top"]
    used = E * (1 - (1 - top / E) ** T)  # experts that some token chooses, about
    weight = 0.5 + 4 / c["group"] if c["bits"] == 4 else 1 + 4 / BLOCK ** 2
    return {"bytes": int(3 * used * H * F * weight) + 2 * E * H + 4 * T * H, "flops": 2 * T * (E * H + 3 * top * H * F)}


# ---- 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["kind"] == "quant":
        rows, K = s["x"].shape
        values = torch.empty(rows, K, dtype=torch.float64, device=DEV)
        scales = torch.empty(-(-rows // c["tile"]), _blocks(K), dtype=torch.float64, device=DEV)
        for b in range(_blocks(K)):
            x = s["x"][:, b * BLOCK:(b + 1) * BLOCK].double()
            top = torch.zeros(scales.shape[0], dtype=torch.float64, device=DEV)
            of = torch.arange(rows, device=DEV) // c["tile"]
            top = top.scatter_reduce(0, of, x.abs().max(1).values, "amax").clamp(min=LEAST)
            v = x * (TOP / top)[of][:, None]
            # three bits behind the leading one, the smallest leading one 2^-6
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
            values[:, b * BLOCK:(b + 1) * BLOCK] = torch.round(v / step) * step
            scales[:, b] = top / TOP
        return values, scales
    if c["kind"] == "gemm":
        out = torch.zeros(c["M"], c["N"], dtype=torch.float64, device=DEV)
        for b in range(_blocks(c["K"])):
            at = slice(b * BLOCK, min(c["K"], (b + 1) * BLOCK))
            rows = torch.arange(c["N"], device=DEV) // BLOCK
            out += (s["a"][:, at].double() * s["sa"][:, b:b + 1].double()) @ (s["w"][:, at].double() * s["sw"][rows, b:b + 1].double()).T
        return out
    T, H, F = c["tokens"], c["hidden"], c["ff"]
    x = s["x"].double()
    score = torch.einsum("th,eh->te", x, s["router"].double())
    p = 1 / (1 + torch.exp(-score)) if c["sigmoid"] else torch.exp(score - score.max(1, keepdim=True).values)
    if not c["sigmoid"]:
        p = p / p.sum(1, keepdim=True)
    ranked = p if s["bias"] is None else p + s["bias"].double()
    out = torch.zeros(T, H, dtype=torch.float64, device=DEV)

    def dense(kept, e):
        if c["bits"] == 8:
            w, scale = kept[0][e].double(), kept[1][e].double()
            rows, cols = torch.arange(w.shape[0], device=DEV) // BLOCK, torch.arange(w.shape[1], device=DEV) // BLOCK
            return w * scale[rows][:, cols]
        words, scale, least = (t[e] for t in kept)
        k = torch.arange(words.shape[1] * 8, device=DEV)
        codes = (words.long()[:, k // 8] >> (4 * (k % 8))) & 15
        return codes.double() * scale.double()[:, k // c["group"]] + least.double()[:, k // c["group"]]

    order = torch.sort(ranked, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    lists = order.tolist()
    for e in sorted({e for row in lists for e in row}):
        up, down = dense(s["up"], e), dense(s["down"], e)
        for t in [t for t, row in enumerate(lists) if e in row]:
            gate, rise = up[:F] @ x[t], up[F:] @ x[t]
            share = p[t, e] / (p[t, order[t]].sum() if c["norm"] else 1.0)
            out[t] += share * (down @ (gate / (1 + torch.exp(-gate)) * rise))
    return out
