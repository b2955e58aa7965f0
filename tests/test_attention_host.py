"""The attention operators without a GPU: the C entries' refusals, the binding's, and the rotary tables."""
import ctypes as C
import inspect
import math

import pytest
import torch

import miori_b200 as mb
from miori_b200 import ops
from miori_b200._lib import lib

OK = 0x1000  # aligned, never dereferenced: validation fails first


def strides(*values):
    return (C.c_int64 * len(values))(*values)


def test_attention_entries_reject_bad_arguments():
    s8, s10 = strides(256, 64, 256, 64, 128, 64, 128, 64), strides(256, 64, 256, 64, 2048, 1024, 64, 2048, 1024, 64)

    def prompt(q=OK, s=s8, cu=OK, requests=1, tokens=4, keys=4, heads=4, kv_heads=2, dim=64, scale=0.125, ws=None, bytes_=0):
        return lib.miori_attention_prompt(q, OK, OK, OK, s, cu, None, requests, tokens, keys, heads, kv_heads, dim, scale, 0, ws, bytes_, None)

    def paged(q=OK, s=s10, table=OK, width=3, pages=3, page=16, heads=4, kv_heads=2, dim=64):
        return lib.miori_attention_paged(q, OK, OK, OK, s, table, OK, OK, 1, 4, width, pages, page, heads, kv_heads, dim, 1, 0.125, 0, None, 0, None)

    for call, text in ((lambda: prompt(q=None), b"null"), (lambda: prompt(cu=None), b"null"), (lambda: prompt(q=OK + 2), b"aligned"),
                       (lambda: prompt(tokens=0), b"empty"), (lambda: prompt(requests=65536), b"65535"), (lambda: prompt(dim=80), b"64 or 128"),
                       (lambda: prompt(heads=5), b"evenly"), (lambda: prompt(heads=130), b"at most 64"), (lambda: prompt(scale=0.0), b"scale"),
                       (lambda: prompt(scale=math.inf), b"scale"), (lambda: prompt(scale=math.nan), b"scale"),
                       (lambda: prompt(s=strides(256, 64, 256, 64, 128, 60, 128, 64)), b"strides"),
                       (lambda: prompt(s=strides(0, 64, 256, 64, 128, 64, 128, 64)), b"strides"), (lambda: prompt(keys=0), b"keys"),
                       (lambda: prompt(ws=OK, bytes_=100), b"workspace"), (lambda: paged(table=None), b"null"), (lambda: paged(width=0), b"empty"),
                       (lambda: paged(page=12), b"power of two"), (lambda: paged(page=4), b"power of two"), (lambda: paged(width=1 << 30), b"2^31")):
        assert call() == -1
        assert text in lib.miori_last_error(), lib.miori_last_error()
    assert lib.miori_attention_workspace_bytes() > 4096


def test_page_and_rope_entries_reject_bad_arguments():
    def slots(held=OK, after=OK + 64, requests=4, width=3, page=16):
        return lib.miori_page_slots(held, OK, OK, OK, OK, OK, OK, OK + 128, after, OK + 256, requests, width, page, 5, 4, 0, None)

    cs = strides(2048, 1024, 64, 2048, 1024, 64)

    def rope(qkv=OK, row=256, cache=cs, tokens=2, heads=2, kv_heads=1, dim=64, rotary=64, axes=1, pages=3, page=16):
        return lib.miori_rope_kv(qkv, row, OK, None, OK, OK, None, None, 0.0, OK, OK, OK, cache, tokens, heads, kv_heads, dim, rotary, axes, pages, page, 0, None)

    for call, text in ((lambda: slots(held=None), b"null"), (lambda: slots(requests=0), b"requests"), (lambda: slots(requests=16385), b"requests"),
                       (lambda: slots(width=0), b"empty"), (lambda: slots(page=0), b"empty"), (lambda: slots(after=OK), b"output"),
                       (lambda: rope(qkv=None), b"null"), (lambda: rope(tokens=0), b"empty"), (lambda: rope(dim=32), b"64 or 128"),
                       (lambda: rope(rotary=24), b"rotary"), (lambda: rope(rotary=80), b"rotary"), (lambda: rope(axes=5), b"axes"),
                       (lambda: rope(row=248), b"rows"), (lambda: rope(row=257), b"rows"), (lambda: rope(qkv=OK + 4), b"aligned"),
                       (lambda: rope(cache=strides(2048, 1024, 60, 2048, 1024, 64)), b"strides"), (lambda: rope(pages=1 << 31, page=2), b"2^31")):
        assert call() == -1
        assert text in lib.miori_last_error(), lib.miori_last_error()


@pytest.mark.parametrize("name", ["page_slots", "rope_kv", "attention_paged", "attention_prompt"])
def test_no_operator_takes_cpu_tensors(name):
    fn = getattr(ops, name)
    numbers = {"page": 16, "tokens": 4, "heads": 2, "max_new": 1}
    need = [p.name for p in inspect.signature(fn).parameters.values() if p.default is p.empty]
    with pytest.raises(ValueError, match="no CPU path"):
        fn(*[numbers.get(n, torch.zeros((16, 64), dtype=torch.bfloat16)) for n in need])


def test_turns_are_whole_parts_of_a_turn():
    turns, axes = mb.rope_turns(64, theta=1e4, sections=(12, 10, 10))
    assert turns.dtype == torch.int64 and axes.tolist() == [0] * 12 + [1] * 10 + [2] * 10
    for j, t in enumerate(turns.tolist()):
        assert abs((t % 2 ** 64) / 2 ** 64 * 2 * math.pi - 1e4 ** (-j / 32)) < 1e-15
    assert mb.rope_turns(16, theta=1e4, sections=(4, 2, 2), interleaved=True)[1].tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    # a frequency of more than a turn a position, and a negative one, keep what is left of a turn
    turns, _ = mb.rope_turns(16, inv_freq=[2 * math.pi * 1.25, -math.pi / 2, 0, 0, 0, 0, 0, 0])
    assert [t % 2 ** 64 for t in turns.tolist()[:2]] == [2 ** 62, 3 * 2 ** 62]
    for bad in ({"rotary": 24, "theta": 1e4}, {"rotary": 64}, {"rotary": 64, "theta": 1e4, "inv_freq": [1.0] * 32}, {"rotary": 64, "inv_freq": [1.0]},
                {"rotary": 64, "theta": 1e4, "sections": (30, 1)}, {"rotary": 64, "theta": 1e4, "sections": (8, 8, 8, 4, 4)}):
        with pytest.raises(ValueError):
            mb.rope_turns(**bad)
