"""Kernels with tensor memory on several streams at once, each behind launches that let it start early: the results of the same calls one at a time."""
import pytest
import torch

import miori_b200 as mb
import test_fp8_gpu as fp8
from miori_b200 import synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def calls():
    """Few rows with K over clusters, tiles on pairs, and the products of the bf16 cache, few rows and many."""
    found = []
    for M, N, K, tune in ((1, 2048, 2048, 0), (20, 1024, 4096, 3 << 20 | 3 << 23), (60, 512, 2048, 3 << 20 | 2 << 23), (5, 4096, 1024, 1 << 20 | 1 << 23), (300, 700, 1500, 5 << 20)):
        ops = fp8.operands(M, N, K, M + N)
        found.append(lambda ops=ops, tune=tune: mb.gemm_fp8(*ops, flags=tune))
    q, s, b = synth.make_weight(2048, 8192, 4, 64, seed=3, device=DEV)
    cache = mb.dequant4_cache(q, s, b, group=64)
    for M in (30, 300):
        x = synth.make_activation(M, 8192, seed=M, device=DEV)
        ws = mb.gemm_workspace(M, 2048, 8192, DEV)
        found.append(lambda x=x, ws=ws: mb.gemm_bf16_cache(x, cache, 2048, flags=mb.LAUNCH_PDL, workspace=ws))
    return found


def test_several_streams_at_once():
    todo = calls()
    want = [call() for call in todo]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in todo]
    for first in range(8):
        got = []
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                # a call in a stream of its own, several times, between calls whose workspace nobody shares
                got.append([todo[i]() for _ in range(1 + (first + i) % 4)])
        torch.cuda.synchronize()
        assert all(torch.equal(t, w) for results, w in zip(got, want) for t in results)
    # one behind the other on one stream: each may begin while the one before drains
    for _ in range(5):
        got = [call() for _ in range(3) for call in todo]
        assert all(torch.equal(t, want[i % len(todo)]) for i, t in enumerate(got))
    assert mb.lib.miori_device_error_poll() == 0
