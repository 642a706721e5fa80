"""MXFP4 operators without a GPU: refusals of the C ABI (nothing is launched), schemas, FakeTensor shapes,
scale layouts and the block's precision argument."""
import ctypes

import numpy as np
import pytest
import torch

import joyomni_ops as jo
from joyomni_ops import mxfp4_linear as ml
from oracle import mxfp4 as mx

lib = jo._LIB
P = [ctypes.c_void_p(0x100000 * (i + 1)) for i in range(10)]


def refused(st, code, fragment):
    assert st == code and fragment in lib.joy_last_error().decode(), lib.joy_last_error()


def test_quant_refusals():
    f = lambda x=P[0], dt=0, ld=256, q=P[1], s=P[2], slab=32, M=4, K=256: (  # noqa: E731
        lib.joy_per_block_quant_mxfp4(x, dt, ld, q, s, slab, M, K, None))
    refused(f(K=48), 1, "multiple of 32")
    refused(f(dt=3), 1, "bfloat16, float16 or float32")
    refused(f(M=-1), 1, "[M, K]")
    refused(f(x=None), 1, "input must be non-null")
    refused(f(x=ctypes.c_void_p(0x1001)), 1, "naturally aligned")
    refused(f(dt=2, x=ctypes.c_void_p(0x1002)), 1, "naturally aligned")
    refused(f(ld=128), 1, "row stride must be >= K")
    refused(f(q=None), 1, "non-null")
    refused(f(s=None), 1, "non-null")
    refused(f(q=ctypes.c_void_p(0x1008)), 2, "16-byte aligned")
    refused(f(s=ctypes.c_void_p(0x1004)), 2, "8-byte aligned")
    refused(f(K=512, ld=512, slab=24), 1, "slab stride")
    refused(f(K=512, ld=512, slab=36), 1, "slab stride")
    refused(f(K=512, ld=512, slab=1 << 31), 2, "2^31 bytes")
    refused(f(M=1 << 28), 2, "2^31 bytes")
    refused(f(q=ctypes.c_void_p(0x100000 + 4 * 512 - 16)), 1, "must not overlap")
    assert f(M=0) == 0 and f(K=0) == 0


def test_dequant_refusals():
    f = lambda q=P[0], s=P[1], slab=32, o=P[2], dt=0, M=4, K=256: (  # noqa: E731
        lib.joy_mxfp4_dequantize(q, s, slab, o, dt, M, K, None))
    refused(f(K=16), 1, "multiple of 32")
    refused(f(dt=9), 1, "out_dtype")
    refused(f(o=None), 1, "out must be non-null")
    refused(f(o=ctypes.c_void_p(0x1008)), 2, "16-byte aligned")
    refused(f(q=None), 1, "non-null")
    refused(f(o=P[0]), 1, "must not overlap")
    assert f(M=0) == 0


def product(name, **kw):
    a = dict(a=P[0], b=P[1], sa=P[2], la=8 * 64, sb=P[3], lb=8 * 64, bias=None, res=P[4], ldr=64, gate=P[5], out=P[6],
             dt=0, q=P[6], s=P[7], ls=8 * 64, M=64, N=64, K=512, epi=0)
    a.update(kw)
    if name == "plain":
        return lib.joy_mxfp4_scaled_mm(a["a"], a["b"], a["sa"], a["la"], a["sb"], a["lb"], a["bias"], a["out"], a["dt"],
                                       a["M"], a["N"], a["K"], a["epi"], None)
    if name == "residual":
        return lib.joy_mxfp4_scaled_mm_gated_residual(a["a"], a["b"], a["sa"], a["la"], a["sb"], a["lb"], a["bias"],
                                                      a["res"], a["ldr"], a["gate"], a["out"], a["dt"], a["M"], a["N"],
                                                      a["K"], None)
    return lib.joy_mxfp4_scaled_mm_gelu_tanh_quant(a["a"], a["b"], a["sa"], a["la"], a["sb"], a["lb"], a["bias"], a["dt"],
                                                   a["q"], a["s"], a["ls"], a["M"], a["N"], a["K"], None)


@pytest.mark.parametrize("name", ["plain", "residual", "quant"])
def test_product_refusals(name):
    f = lambda **kw: product(name, **kw)  # noqa: E731
    refused(f(K=40), 1, "multiple of 32")
    refused(f(K=0), 1, "K must be positive")
    refused(f(M=-1), 1, "cannot be multiplied")
    refused(f(dt=2), 1, "Half or BFloat16")
    refused(f(a=None), 1, "mat_a codes and scales must be non-null")
    refused(f(sb=None), 1, "mat_b codes and scales must be non-null")
    refused(f(b=ctypes.c_void_p(0x1008)), 2, "16-byte aligned")
    refused(f(sa=ctypes.c_void_p(0x1004)), 2, "8-byte aligned")
    refused(f(la=8), 1, "mat_a slab stride")
    refused(f(lb=8 * 64 + 4), 1, "mat_b slab stride")
    refused(f(bias=ctypes.c_void_p(0x1008)), 2, "bias must be 16-byte aligned")
    refused(f(N=1 << 22), 2, "2^22")
    refused(f(K=1 << 22), 2, "2^22")
    refused(f(M=1 << 27, la=8 << 27, K=256, N=1 << 16, lb=8 << 16), 2, "tiles")
    refused(f(a=P[6]), 1, "must not overlap")
    refused(f(b=ctypes.c_void_p(0x100000 * 7 + 16)), 1, "must not overlap")
    assert f(M=0) == 0 and f(N=0) == 0
    if name == "quant":
        refused(f(N=72), 1, "N must be a multiple of 32")
        refused(f(q=None), 1, "out must be non-null")
        refused(f(s=None), 1, "output codes and scales must be non-null")
        refused(f(s=P[2]), 1, "must not be the operands'")
        refused(f(N=512, lb=8 * 512, ls=8), 1, "output slab stride")
    else:
        refused(f(N=68), 1, "multiple of 16 bytes")
        refused(f(out=ctypes.c_void_p(0x1008)), 2, "out must be 16-byte aligned")
        refused(f(out=None), 1, "out must be non-null")
    if name == "plain":
        refused(f(epi=2), 1, "unknown epilogue")
    if name == "residual":
        refused(f(res=None), 1, "residual and gate must be non-null")
        refused(f(gate=None), 1, "residual and gate must be non-null")
        refused(f(ldr=32), 1, "row stride must be >= N")
        refused(f(ldr=68), 2, "16-byte aligned")
        refused(f(ldr=1 << 22), 2, "2^22")
        refused(f(gate=ctypes.c_void_p(0x1002)), 2, "16-byte aligned")
        refused(f(res=P[6], ldr=72), 1, "in-place residual")
        refused(f(res=ctypes.c_void_p(0x100000 * 7 + 64)), 1, "not overlap it")


def test_norm_refusals():
    f = lambda x=P[0], ld=64, dt=0, sc=P[1], sh=P[2], rows=1, q=P[3], s=P[4], M=4, N=64, nt=0: (  # noqa: E731
        lib.joy_fused_norm_scale_shift_mxfp4(x, ld, dt, None, None, sc, sh, rows, q, s, 8 * M, M, N, nt, 1e-6, None))
    refused(f(N=48), 1, "multiple of 32")
    refused(f(rows=2), 1, "scale/shift rows")
    refused(f(nt=2), 1, "norm_type")
    refused(f(dt=4), 1, "Unsupported dtype")
    refused(f(ld=32), 1, "x row stride")
    refused(f(sc=None), 1, "non-null")
    refused(f(sh=ctypes.c_void_p(0x1001)), 1, "naturally aligned")
    refused(f(q=None), 1, "non-null")
    assert f(M=0, rows=1) == 0


def test_overlaps_are_refused():
    """An output over bytes that other workgroups still read: operands, scales, vectors, or its own scales."""
    v = ctypes.c_void_p
    quant = lambda x, q, s: lib.joy_per_block_quant_mxfp4(x, 0, 512, q, s, 32, 4, 512, None)  # noqa: E731
    refused(quant(P[0], P[1], v(P[0].value + 4000)), 1, "must not overlap")  # input: 4096 bytes
    refused(quant(P[0], P[1], v(P[1].value + 1016)), 1, "must not overlap")  # codes: 1024
    refused(lib.joy_mxfp4_dequantize(P[0], P[1], 32, v(P[1].value + 48), 0, 4, 512, None), 1, "must not overlap")
    for name in ("plain", "residual", "quant"):
        for at in (P[2].value + 1008, P[3].value, P[8].value + 112):
            at = v(at)
            refused(product(name, bias=P[8], out=at, q=at), 1, "out must not overlap the scales or the bias")
    refused(product("residual", out=v(P[5].value + 112)), 1, "out must not overlap gate")
    for at in (P[0].value + 64 * 256 - 8, P[1].value, P[2].value + 1016, P[3].value, P[6].value + 64 * 32 - 8, P[8].value):
        refused(product("quant", bias=P[8], s=v(at)), 1, "output scales must not be")
    norm = lambda q, s: lib.joy_fused_norm_scale_shift_mxfp4(  # noqa: E731
        P[0], 64, 0, P[5], P[6], P[1], P[2], 1, q, s, 32, 4, 64, 0, 1e-6, None)
    for i, size in ((0, 512), (1, 128), (2, 128), (5, 128), (6, 128), (3, 128)):
        refused(norm(P[3], v(P[i].value + size - 8)), 1, "must not overlap")
        if i != 3:
            refused(norm(v(P[i].value + size - 16), P[4]), 1, "must not overlap")


def test_cpu_tensors_have_no_kernel():
    q, s = ml.empty_mxfp4(4, 64, "cpu")
    with pytest.raises(NotImplementedError):
        jo.per_block_quant_mxfp4(torch.zeros(4, 64), q, s)
    with pytest.raises(NotImplementedError):
        jo.mxfp4_scaled_mm(q, q.t(), s, s, torch.bfloat16)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *n, dt=torch.uint8: torch.empty(*n, dtype=dt, device="cuda")  # noqa: E731
        a, w, sa, sw = e(300, 256), e(1024, 256), e(2, 300, 8), e(2, 1024, 8)
        assert jo.mxfp4_scaled_mm(a, w.t(), sa, sw, torch.float16).shape == (300, 1024)
        assert jo.mxfp4_scaled_mm_gelu_tanh(a, w.t(), sa, sw, torch.bfloat16).dtype == torch.bfloat16
        r = e(300, 1024, dt=torch.bfloat16)
        assert jo.mxfp4_scaled_mm_gated_residual(a, w.t(), sa, sw, r, r[0]).shape == r.shape
        assert jo.mxfp4_scaled_mm_gated_residual(a, w.t(), sa, sw, r, r[0], inplace=True) is r
        assert jo.mxfp4_dequantize(a, sa, torch.float32).shape == (300, 512)
        jo.per_block_quant_mxfp4(e(300, 512, dt=torch.float32), a, sa)
        jo.mxfp4_scaled_mm_gelu_tanh_quant(a, w.t(), sa, sw, None, e(300, 512), e(4, 300, 8))
        x = e(300, 512, dt=torch.bfloat16)
        jo.fused_norm_scale_shift_mxfp4(x, None, None, x[:1], x[:1], "layer", 1e-6, a, sa)


def test_outputs_are_declared_mutable():
    for name, outs in (("per_block_quant_mxfp4", ["output_q", "output_s"]),
                       ("mxfp4_scaled_mm_gelu_tanh_quant", ["output_q", "output_s"]),
                       ("fused_norm_scale_shift_mxfp4", ["output_q", "output_s"]),
                       ("mxfp4_scaled_mm_gated_residual_", ["residual"])):
        args = getattr(torch.ops.joyomni_ops, name).default._schema.arguments
        assert [a.name for a in args if a.alias_info is not None and a.alias_info.is_write] == outs


def test_scale_layout_conversions():
    s = np.random.default_rng(0).integers(1, 255, (7, 19)).astype(np.uint8)
    t = ml.scales_from_row_major(torch.from_numpy(s))
    assert t.dtype == torch.float8_e8m0fnu and np.array_equal(t.view(torch.uint8).numpy(), mx.slabs(s))
    assert np.array_equal(ml.scales_to_row_major(t, 19 * 32).view(torch.uint8).numpy(), s)
    with pytest.raises(ValueError, match="one byte"):
        ml.scales_from_row_major(torch.zeros(3, 4))
    with pytest.raises(ValueError, match="multiple of 32"):
        ml.empty_mxfp4(4, 40, "cpu")


def test_block_precision_argument():
    from joyomni_ops.dit_block import QuantizedDoubleStreamBlock
    with pytest.raises(ValueError, match="precision must be"):
        QuantizedDoubleStreamBlock(64, 1, 64, "cpu", torch.Generator(), precision="int4")


def test_inplace_residual_alignment():
    """In place, a residual that is not 16-byte aligned is refused (out of place the operator copies it)."""
    at = ctypes.c_void_p(P[6].value + 8)
    refused(product("residual", res=at, out=at), 2, "16-byte aligned")
    assert "16-byte aligned" in jo.mxfp4_scaled_mm_gated_residual.__doc__
