"""GPU: the adaLN norm with MXFP4 output where its kernels change (8192 and 16384 values a row), and with gamma alone."""
import pytest
import torch

from gpu_util import DEV, announce, gen, kernels_of, outlier_acts
from test_gpu_mxfp4 import TYPES, host, room
from test_gpu_mxfp4 import test_norm_mxfp4 as norm_case  # (M, N, kind, dtype): against the 64-bit oracle

pytestmark = pytest.mark.gpu


# values a row, kernel of aligned rows with an affine part: vectors a lane, or the general kernel's
ROUTES = [(2048, "_rows<{}, {}, 1, true>"), (2080, "_rows<{}, {}, 2, true>"), (8192, "_rows<{}, {}, 2, true>"),
          (8224, "_rows<{}, {}, 4, true>"), (16384, "_rows<{}, {}, 4, true>"), (16416, "<{}, {}, true>")]


@pytest.mark.parametrize("N,kernel", ROUTES)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_gamma_alone(N, kernel, dtype):
    """gamma without beta: as with a beta of zeros, bit for bit; RMS ignores beta."""
    import joyomni_ops as jo
    announce("fused_norm_scale_shift_mxfp4 gamma alone", N, dtype)
    M, t, g = 5, TYPES[dtype], gen(N)
    x = outlier_acts(M, N, g).to(t).to(DEV)
    gamma, beta, scale, shift = ((c + 0.3 * torch.randn(N, generator=g)).to(t).to(DEV) for c in (1, 0, 0, 0))
    for nt, kind in enumerate(("layer", "rms")):
        def run(b, x=x):
            q, s = room(M, N)
            jo.fused_norm_scale_shift_mxfp4(x, gamma, b, scale[None], shift[None], kind, 1e-6, q, s)
            return host(q), host(s)

        alone, names = kernels_of(lambda: run(None))
        if names:
            assert "norm_mod_mxfp4" + kernel.format(list(TYPES).index(dtype), nt) in names, names
        zeros = run(torch.zeros_like(beta))
        assert (alone[0] == zeros[0]).all() and (alone[1] == zeros[1]).all()
        other = run(beta)
        same = (alone[0] == other[0]).all() and (alone[1] == other[1]).all()
        assert same == (kind == "rms")
        odd = torch.zeros(M, N + 8, dtype=t, device=DEV)  # unaligned rows: the general kernel, element by element
        odd[:, 1: 1 + N] = x
        one, names = kernels_of(lambda: run(None, odd[:, 1: 1 + N]))
        if names:
            assert f"norm_mod_mxfp4<{list(TYPES).index(dtype)}, {nt}, false>" in names, names
        zero = run(torch.zeros_like(beta), odd[:, 1: 1 + N])
        assert (one[0] == zero[0]).all() and (one[1] == zero[1]).all()


@pytest.mark.parametrize("M,N", [(3, 8224), (2, 16384), (3, 16416)])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_long_rows(M, N, kind, dtype):
    norm_case(M, N, kind, dtype)
