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
