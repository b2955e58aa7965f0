"""The tensor-level operators over the C ABI.  torch is used for device memory and streams only; every
computation happens in libmiori_b200.so.

The operators themselves are C functions (csrc/binding.cpp, built as _native.so): each checks its
tensors, allocates the output when none is given and enqueues on the current stream.  An operator's
device work is a few microseconds, so the call path is native as well.  As with the library there is
no fallback: without _native.so this module does not import.
"""
from __future__ import annotations

import math

import torch

from ._lib import MioriError, check, lib
from . import _native

_native.bind(lib._handle, MioriError)

from ._native import (argmax, attention_paged, attention_prompt, dequant4_cache, dequant4_rowmajor, dequant8_rowmajor, embed8,  # noqa: E402,F401
                      gemm_bf16_cache, gemm_bf16_strided, gemm_fp8, gemv4, gemv4_post_norm_add, gemv4_rmsnorm,
                      gemv4_rmsnorm_silu, gemv4_silu, gemv8, gemv8_rmsnorm, gemv_bf16_cache, linear4,
                      moe4, moe_fp8, page_slots, post_norm_add, quant_fp8, rmsnorm, rope_kv, silu_mul)


def cache_to_rowmajor(cache, N, K):
    """The row-major [N][K] tensor behind a cache of dequant4_cache."""
    if not cache.is_cuda:
        raise ValueError("miori_b200 ops need CUDA tensors (there is no CPU path)")
    if not cache.is_contiguous():
        raise ValueError("miori_b200 ops need contiguous tensors")
    o = torch.empty((N, K), dtype=torch.bfloat16, device=cache.device)
    check(lib.miori_cache_to_rowmajor(cache.data_ptr(), o.data_ptr(), N, K, torch.cuda.current_stream().cuda_stream))
    return o


def gemm_workspace(M, N, K, device):
    """Scratch tensor of the size miori_gemm_workspace_bytes recommends, or None."""
    nbytes = lib.miori_gemm_workspace_bytes(M, N, K)
    return torch.empty(nbytes // 4, dtype=torch.float32, device=device) if nbytes else None


def attention_workspace(device):
    """Zeroed scratch tensor for attention_paged and attention_prompt: one per stream that may run them."""
    return torch.zeros(lib.miori_attention_workspace_bytes(), dtype=torch.uint8, device=device)


def moe_workspace(tokens, top, ff, device):
    """Scratch tensor for moe4 and moe_fp8 of up to `tokens` tokens: one per stream that may run them."""
    return torch.empty(lib.miori_moe_workspace_bytes(tokens, top, ff), dtype=torch.uint8, device=device)


def rope_turns(rotary, theta=None, sections=None, interleaved=False, inv_freq=None, device=None):
    """(turns, axes) tensors of rope_kv for `rotary` dimensions, made once.

    Pair j turns by theta ** (-2 j / rotary) radians a position, or by inv_freq[j] where a sequence is given (scaled or
    trained frequencies).  `sections`: pairs of each axis, in the order of the axes (their sum is rotary / 2); one after
    the other, or with `interleaved` dealt out in turns, an axis dropping out when it has its number.  None: one axis."""
    half = rotary // 2
    if rotary <= 0 or rotary % 16:
        raise ValueError("rotary dimensions are a multiple of 16")
    if (theta is None) == (inv_freq is None):
        raise ValueError("one of theta and inv_freq is needed")
    freq = [float(f) for f in inv_freq] if inv_freq is not None else [float(theta) ** (-2.0 * j / rotary) for j in range(half)]
    if len(freq) != half:
        raise ValueError(f"{half} frequencies expected, got {len(freq)}")
    sections = [half] if sections is None else [int(n) for n in sections]
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != half:
        raise ValueError(f"sections are one to four numbers of pairs with the sum {half}, got {sections}")
    if interleaved:
        left, order = list(sections), []
        while len(order) < half:
            for a in range(len(left)):
                if left[a]:
                    left[a] -= 1
                    order.append(a)
    else:
        order = [a for a, n in enumerate(sections) for _ in range(n)]
    # an angle as a whole number of 2^-64 turns, modulo one turn; int64 holds the bits of the unsigned number
    units = [round(math.fmod(f / (2.0 * math.pi), 1.0) * 2.0 ** 64) % 2 ** 64 for f in freq]
    turns = torch.tensor([u - 2 ** 64 if u >= 2 ** 63 else u for u in units], dtype=torch.int64, device=device)
    return turns, torch.tensor(order, dtype=torch.int32, device=device)
