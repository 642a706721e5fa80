"""GPU: the MXFP4 product's tile kernels where a workgroup takes several tiles, against the 64-bit oracle with
test_gpu_mxfp4.py's tolerances, the route of each call held by kernel name (256 CUs)."""
import pytest
import torch

from gpu_util import DEV, announce, kernels_of
from oracle import mxfp4 as mx
from test_gpu_mxfp4 import TYPES, check_mx, check_rounded, gelu_tol, host, problem, room, sums

pytestmark = pytest.mark.gpu


def expect(names, kernel, epi):
    if torch.cuda.get_device_properties(0).multi_processor_count == 256 and names:
        assert any(f"mxfp4_gemm_{kernel.format(epi)}" == n for n in names), (kernel, epi, names)


# One slab a tile, several tiles a workgroup: 344 tiles of 128 x 192, 511 of 128 x 128, 387 of 128 x 256 and, with 256 x
# 256 tiles, 129 and 20 rest tiles of 64 x 256 on 127 and 16 workgroups. Bias and gate differ from column to column, so
# that those of another tile show.
SINGLE_SLAB = [(129, 32896, 256, "bf16", "tiles<{}, {}, 2, 3, 0>"), (129, 32896, 32, "fp16", "tiles<{}, {}, 2, 3, 0>"),
               (800, 9344, 256, "fp16", "tiles<{}, {}, 2, 2, 0>"), (800, 9344, 32, "bf16", "tiles<{}, {}, 2, 2, 0>"),
               (373, 32896, 32, "bf16", "tiles<{}, {}, 2, 4, 0>"),
               (312, 32896, 256, "bf16", "tiles<{}, {}, 4, 4, 1>"), (312, 32896, 32, "fp16", "tiles<{}, {}, 4, 4, 1>"),
               (3120, 5120, 256, "fp16", "tiles<{}, {}, 4, 4, 1>"), (3120, 5120, 32, "bf16", "tiles<{}, {}, 4, 4, 1>")]


@pytest.mark.parametrize("M,N,K,dtype,kernel", SINGLE_SLAB)
def test_single_slab_tiles(M, N, K, dtype, kernel):
    import joyomni_ops as jo
    announce("mxfp4 one slab, several tiles", M, N, K, dtype)
    a, w, sa, sw, va, vw, bias, res, gate = problem(M, N, K, dtype, M + K)
    kernel = kernel.replace("{}", str(dtype == "bf16").lower(), 1)
    y, tol = sums(va, vw, bias)
    t, b, g, w = TYPES[dtype], bias.to(DEV), gate.to(DEV), w.t()
    out, names = kernels_of(lambda: jo.mxfp4_scaled_mm(a, w, sa, sw, t, b))
    expect(names, kernel, 0)
    check_rounded(out, y, tol, dtype)
    out, names = kernels_of(lambda: jo.mxfp4_scaled_mm_gelu_tanh(a, w, sa, sw, t, b))
    expect(names, kernel, 1)
    z, ztol = mx.gelu_tanh(y), gelu_tol(y, tol)
    check_rounded(out, z, ztol, dtype)
    rd = res.to(DEV)
    out, names = kernels_of(lambda: jo.mxfp4_scaled_mm_gated_residual(a, w, sa, sw, rd, g, b))
    expect(names, kernel, 2)
    g64, r64 = gate.double().numpy(), res.double().numpy()
    check_rounded(out, r64 + y * g64, abs(g64) * tol + 2.0 ** -23 * (abs(r64) + abs(y * g64)), dtype)
    jo.mxfp4_scaled_mm_gated_residual(a, w, sa, sw, rd, g, b, inplace=True)
    assert torch.equal(rd, out)
    q, s = room(M, N)
    _, names = kernels_of(lambda: jo.mxfp4_scaled_mm_gelu_tanh_quant(a, w, sa, sw, b, q, s))
    expect(names, kernel, 3)
    check_mx(q, s, z, ztol)
    for _ in range(3):  # again, behind other calls: the same bits
        q2, s2 = room(M, N)
        jo.mxfp4_scaled_mm_gelu_tanh_quant(a, w, sa, sw, b, q2, s2)
        assert (host(q2) == host(q)).all() and (host(s2) == host(s)).all()


@pytest.mark.parametrize("M,N,kernel", [(347, 2080, "tiles<true, {}, 1, 2, 0>"), (701, 4096, "tiles<true, {}, 2, 2, 0>"),
                                        (347, 14400, "tiles<true, {}, 2, 3, 0>"), (347, 16384, "tiles<true, {}, 2, 4, 0>"),
                                        (3121, 5120, "tiles<true, {}, 4, 4, 1>")])
def test_tiles_on_operand_views(M, N, kernel):
    """Rows from an odd one on of larger operands and outputs (scale bases at 8 of 16 bytes, slabs further apart than their
    rows), a residual whose rows are apart: each result, and the rows around the outputs as they were."""
    import joyomni_ops as jo
    announce("mxfp4 tiles on views", M, N)
    K = 544  # the last slab has one block
    a, w, sa, sw, va, vw, bias, res, gate = problem(M + 9, N + 16, K, "bf16", M)
    rows, cols = slice(5, 5 + M), slice(3, 3 + N)
    a, sa, w, sw = a[rows], sa[:, rows], w[cols].t(), sw[:, cols]
    b, g = bias[cols].to(DEV), gate[cols].to(DEV)
    y, tol = sums(va[rows], vw[cols], bias[cols])
    out, names = kernels_of(lambda: jo.mxfp4_scaled_mm(a, w, sa, sw, torch.bfloat16, b))
    expect(names, kernel, 0)
    check_rounded(out, y, tol, "bf16")
    z, ztol = mx.gelu_tanh(y), gelu_tol(y, tol)
    check_rounded(jo.mxfp4_scaled_mm_gelu_tanh(a, w, sa, sw, torch.bfloat16, b), z, ztol, "bf16")
    r = res.to(DEV)[rows, 8: 8 + N]
    assert r.stride(0) == N + 16
    g64, r64 = gate[cols].double().numpy(), res[rows, 8: 8 + N].double().numpy()
    out, names = kernels_of(lambda: jo.mxfp4_scaled_mm_gated_residual(a, w, sa, sw, r, g, b))
    expect(names, kernel, 2)
    check_rounded(out, r64 + y * g64, abs(g64) * tol + 2.0 ** -23 * (abs(r64) + abs(y * g64)), "bf16")
    q, s = room(M + 4, N)
    _, names = kernels_of(lambda: jo.mxfp4_scaled_mm_gelu_tanh_quant(a, w, sa, sw, b, q[1: 1 + M], s[:, 1: 1 + M]))
    expect(names, kernel, 3)
    check_mx(q[1: 1 + M], s[:, 1: 1 + M].contiguous(), z, ztol)
    for t in (q[:1], q[1 + M:], s[:, :1], s[:, 1 + M:]):
        assert (t == 0x5a).all()


def test_inplace_residual_alignment():
    """A contiguous residual at an odd address: copied out of place, refused in place and then as it was."""
    import joyomni_ops as jo
    M, N, K = 9, 64, 64
    a, w, sa, sw, _, _, bias, res, gate = problem(M, N, K, "bf16", 1)
    odd = torch.zeros(M * N + 1, dtype=torch.bfloat16, device=DEV)[1:].view(M, N)
    odd.copy_(res)
    args = (a, w.t(), sa, sw)
    want = jo.mxfp4_scaled_mm_gated_residual(*args, res.to(DEV), gate.to(DEV), bias.to(DEV))
    assert torch.equal(jo.mxfp4_scaled_mm_gated_residual(*args, odd, gate.to(DEV), bias.to(DEV)), want)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        jo.mxfp4_scaled_mm_gated_residual(*args, odd, gate.to(DEV), bias.to(DEV), inplace=True)
    assert torch.equal(odd.cpu(), res)
