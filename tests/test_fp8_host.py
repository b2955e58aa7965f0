"""The operators in 8-bit floating point and the layers of experts without a GPU: the C entries' refusals and the binding's."""
import inspect
import math

import pytest
import torch

import miori_b200 as mb
from miori_b200 import ops
from miori_b200._lib import lib

OK = 0x1000  # aligned, never dereferenced: validation fails first


def refused(call, text):
    assert call() == -1
    assert text in lib.miori_last_error(), lib.miori_last_error()


def test_quant_refuses_bad_arguments():
    def quant(x=OK, x_row=256, q=OK, q_row=256, s=OK, s_row=2, s_col=1, rows=4, K=256, tile=1, flags=0):
        return lib.miori_quant_fp8(x, x_row, q, q_row, s, s_row, s_col, rows, K, tile, flags, None)

    for call, text in ((lambda: quant(x=None), b"null"), (lambda: quant(q=None), b"null"), (lambda: quant(s=None), b"null"),
                       (lambda: quant(rows=0), b"empty"), (lambda: quant(K=0), b"empty"), (lambda: quant(tile=64), b"1 or 128"),
                       (lambda: quant(tile=0), b"1 or 128"), (lambda: quant(x_row=255), b"pitch"), (lambda: quant(x_row=-256), b"pitch"),
                       (lambda: quant(q_row=240), b"pitch"), (lambda: quant(q_row=264), b"16-byte"), (lambda: quant(q=OK + 8), b"16-byte"),
                       (lambda: quant(x=OK + 1), b"aligned"), (lambda: quant(x=OK + 2, flags=64), b"aligned"), (lambda: quant(s=OK + 2), b"aligned"),
                       (lambda: quant(x_row=1 << 41), b"pitch"), (lambda: quant(s_row=1 << 41), b"strides"), (lambda: quant(s_col=-(1 << 41)), b"strides"),
                       (lambda: quant(s_row=0), b"on one another"), (lambda: quant(s_col=0), b"on one another"), (lambda: quant(rows=0x80000000), b"2^31"), (lambda: quant(rows=1 << 30, K=256), b"blocks")):
        refused(call, text)


def test_gemm_refuses_bad_arguments():
    def gemm(a=OK, lda=256, sa=OK, sa_s=(2, 1), w=OK, ldw=256, sw=OK, sw_s=(2, 1), C=OK, ldc=64, M=4, N=64, K=256, flags=0):
        return lib.miori_gemm_fp8(a, lda, sa, *sa_s, w, ldw, sw, *sw_s, C, ldc, M, N, K, flags, None)

    for call, text in ((lambda: gemm(a=None), b"null"), (lambda: gemm(sa=None), b"null"), (lambda: gemm(w=None), b"null"), (lambda: gemm(sw=None), b"null"),
                       (lambda: gemm(C=None), b"null"), (lambda: gemm(M=0), b"empty"), (lambda: gemm(N=0), b"empty"), (lambda: gemm(K=0), b"empty"),
                       (lambda: gemm(a=OK + 8), b"16-byte"), (lambda: gemm(w=OK + 4), b"16-byte"), (lambda: gemm(lda=264), b"16-byte"), (lambda: gemm(ldw=260), b"16-byte"),
                       (lambda: gemm(lda=240), b"pitch"), (lambda: gemm(ldw=128), b"pitch"), (lambda: gemm(ldc=63), b"pitch"), (lambda: gemm(ldc=-64), b"pitch"),
                       (lambda: gemm(sa_s=(1 << 41, 1)), b"strides"), (lambda: gemm(sw_s=(1, 1 << 50)), b"strides"), (lambda: gemm(C=OK + 2), b"aligned"),
                       (lambda: gemm(C=OK + 1, flags=1), b"aligned"), (lambda: gemm(sa=OK + 2), b"aligned"), (lambda: gemm(sw=OK + 1), b"aligned"),
                       (lambda: gemm(M=0x7FFFFFFF), b"2^31"), (lambda: gemm(K=16385, lda=16400, ldw=16400, flags=2 << 20), b"16384")):
        refused(call, text)


def test_layers_of_experts_refuse_bad_arguments():
    size = lib.miori_moe_workspace_bytes(4, 2, 256)
    assert lib.miori_moe_workspace_bytes(5, 2, 256) - size == 2 * 256 * 4  # fp32 activations of each pair of a token and an expert

    def both(text, step=True, **kw):
        d = dict(x=OK, router=OK, bias=None, up=OK, su=OK, bu=OK, down=OK, sd=OK, bd=OK, out=OK, tokens=4, experts=8, top=2, hidden=256, ff=256, group=64,
                 factor=1.0, flags=0, ws=OK, bytes_=1 << 20)
        d.update(kw)
        tail = (d["factor"], d["flags"], d["ws"], d["bytes_"], None)
        sizes = tuple(d[k] for k in ("out", "tokens", "experts", "top", "hidden", "ff"))
        refused(lambda: lib.miori_moe4(d["x"], d["router"], d["bias"], d["up"], d["su"], d["bu"], d["down"], d["sd"], d["bd"], *sizes, d["group"], *tail), text)
        if "group" not in kw and "bu" not in kw and "bd" not in kw and step:
            refused(lambda: lib.miori_moe_fp8(d["x"], d["router"], d["bias"], d["up"], d["su"], d["down"], d["sd"], *sizes, *tail), text)

    for name in ("x", "router", "up", "su", "bu", "down", "sd", "bd", "out", "ws"):
        both(b"null", **{name: None})
        both(b"aligned", **{name: OK + 8})
    both(b"aligned", bias=OK + 2)
    both(b"tokens", tokens=0)
    both(b"tokens", tokens=33)
    both(b"experts", experts=0)
    both(b"experts", experts=257)
    both(b"for a token", top=0)
    both(b"for a token", top=9)
    both(b"for a token", top=17, experts=64)
    both(b"multiples", hidden=0)
    both(b"multiples", ff=0)
    both(b"multiples", hidden=250)
    both(b"multiples", ff=264)
    both(b"multiples of 128", hidden=272, step=False)
    both(b"at most", hidden=7296)
    both(b"at most", ff=65664)
    both(b"group", group=128)
    both(b"factor", factor=math.nan)
    both(b"factor", factor=-math.inf)
    both(b"workspace", bytes_=size - 1)


def test_signatures():
    assert str(inspect.signature(mb.quant_fp8)) == "(x, tile=1, flags=0, out=None, scales=None)"
    assert str(inspect.signature(mb.gemm_fp8)) == "(a, sa, w, sw, flags=0, out=None)"
    assert str(inspect.signature(mb.moe4)) == "(x, router, q_up, s_up, b_up, q_down, s_down, b_down, top, workspace, bias=None, group=32, factor=1.0, flags=0, out=None)"
    assert str(inspect.signature(mb.moe_fp8)) == "(x, router, w_up, s_up, w_down, s_down, top, workspace, bias=None, factor=1.0, flags=0, out=None)"


@pytest.mark.parametrize("name", ["quant_fp8", "gemm_fp8", "moe4", "moe_fp8"])
def test_no_cpu_tensors(name):
    t = torch.zeros((16, 64), dtype=torch.bfloat16)
    need = [p for p in inspect.signature(getattr(ops, name)).parameters.values() if p.default is p.empty]
    with pytest.raises(ValueError, match="no CPU path"):
        getattr(ops, name)(*[2 if p.name == "top" else t for p in need])


def fakes():
    """CUDA tensors without memory."""
    from torch._subclasses import FakeTensorMode
    f8 = torch.float8_e4m3fn
    with FakeTensorMode():
        def cuda(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device="cuda")
        return {"x": cuda(4, 256), "half": cuda(4, 256, dtype=torch.float16), "xt": cuda(256, 4).T, "a": cuda(4, 256, dtype=f8), "at": cuda(256, 4, dtype=f8).T,
                "sa": cuda(4, 2), "w": cuda(300, 256, dtype=f8), "sw": cuda(3, 2), "short": cuda(300, 128, dtype=f8), "out": cuda(4, 300), "out16": cuda(4, 300, dtype=torch.bfloat16),
                "xb": cuda(4, 256, dtype=torch.bfloat16), "router": cuda(8, 256, dtype=torch.bfloat16), "bias": cuda(7), "ws": cuda(1 << 20, dtype=torch.uint8),
                "up": cuda(8, 512, 256, dtype=f8), "su": cuda(8, 4, 2), "down": cuda(8, 256, 256, dtype=f8), "sd": cuda(8, 2, 2),
                "q": cuda(8, 512, 32, dtype=torch.int32), "s": cuda(8, 512, 4, dtype=torch.bfloat16), "qd": cuda(8, 256, 32, dtype=torch.int32),
                "ds": cuda(8, 256, 4, dtype=torch.bfloat16), "odd": cuda(8, 513, 256, dtype=f8)}


def test_tensors_of_other_shapes_and_types():
    f = fakes()

    def case(error, match, fn, *args, **kw):
        with pytest.raises(error, match=match):
            fn(*[f[a] if isinstance(a, str) else a for a in args], **{k: f[v] if isinstance(v, str) else v for k, v in kw.items()})

    case(TypeError, "fp32 or bf16", ops.quant_fp8, "half")
    case(ValueError, "contiguous rows", ops.quant_fp8, "xt")
    case(ValueError, "1 or 128", ops.quant_fp8, "x", tile=64)
    case(TypeError, "float8_e4m3fn", ops.quant_fp8, "x", out="x")
    case(ValueError, "shape of x", ops.quant_fp8, "x", out="w")
    case(ValueError, r"scales: \[4\]\[2\]", ops.quant_fp8, "x", out="a", scales="sw")
    case(TypeError, "float8_e4m3fn", ops.gemm_fp8, "x", "sa", "w", "sw")
    case(ValueError, "contiguous", ops.gemm_fp8, "at", "sa", "w", "sw")
    case(ValueError, "rows of 256", ops.gemm_fp8, "a", "sa", "short", "sw")
    case(ValueError, r"sa: \[4\]\[2\]", ops.gemm_fp8, "a", "sw", "w", "sw")
    case(ValueError, r"sw: \[3\]\[2\]", ops.gemm_fp8, "a", "sa", "w", "sa")
    case(ValueError, "output's type", ops.gemm_fp8, "a", "sa", "w", "sw", out="out16")
    case(ValueError, "output's type", ops.gemm_fp8, "a", "sa", "w", "sw", out="x")
    fp8 = ("up", "su", "down", "sd")
    case(TypeError, "bf16", ops.moe_fp8, "x", "router", *fp8, 2, "ws")
    case(ValueError, "bias", ops.moe_fp8, "xb", "router", *fp8, 2, "ws", bias="bias")
    case(ValueError, "2 ff", ops.moe_fp8, "xb", "router", "odd", "su", "down", "sd", 2, "ws")
    case(ValueError, r"w_down: \[8\]\[256\]\[256\]", ops.moe_fp8, "xb", "router", "up", "su", "up", "sd", 2, "ws")
    case(TypeError, "another type", ops.moe_fp8, "xb", "router", "up", "s", "down", "sd", 2, "ws")
    case(ValueError, "group", ops.moe4, "xb", "router", "q", "s", "s", "qd", "ds", "ds", 2, "ws", group=48)
    case(ValueError, "s_up", ops.moe4, "xb", "router", "q", "s", "s", "qd", "ds", "ds", 2, "ws")  # scales of groups of 64 where 32 are meant


def test_tensors_of_several_devices():
    """Refused before anything is launched."""
    f = fakes()
    from torch._subclasses import FakeTensorMode
    with FakeTensorMode():
        far = torch.empty((4, 256), dtype=torch.float8_e4m3fn, device="cuda:1")
        far_ws, far_out = torch.empty(1 << 20, dtype=torch.uint8, device="cuda:1"), torch.empty((4, 2), device="cuda:1")
    fp8 = [f[k] for k in ("up", "su", "down", "sd")]
    for call in (lambda: ops.quant_fp8(f["x"], out=far), lambda: ops.quant_fp8(f["x"], out=f["a"], scales=far_out), lambda: ops.gemm_fp8(far, f["sa"], f["w"], f["sw"]),
                 lambda: ops.moe_fp8(f["xb"], f["router"], *fp8, 2, far_ws)):
        with pytest.raises((ValueError, RuntimeError), match="one device|storage"):
            call()


def test_weights_of_experts_are_contiguous():
    f = fakes()
    from torch._subclasses import FakeTensorMode
    with FakeTensorMode():
        turned = torch.empty((8, 256, 512), dtype=torch.float8_e4m3fn, device="cuda").transpose(1, 2)
    with pytest.raises(ValueError, match="contiguous"):
        ops.moe_fp8(f["xb"], f["router"], turned, f["su"], f["down"], f["sd"], 2, f["ws"])
