"""fp32 arguments of the block-scaled and layer-norm entry points at addresses that are no multiple of four: refused before
any CUDA call."""
import ctypes

import pytest

from float8_experimental_b200 import _native as N

vp = ctypes.c_void_p
P, ODD, ALIGNMENT = vp(256), vp(258), -2


@pytest.mark.parametrize("name", ["mean", "rstd"])
def test_layer_norm_statistics(name):
    stats = {"mean": P, "rstd": P, name: ODD}
    lib = N.load()
    assert lib.f8b200_layer_norm(P, 0, 4, 8, 8, None, None, 0, 1e-5, P, 8, stats["mean"], stats["rstd"], None) == ALIGNMENT
    assert lib.f8b200_layer_norm_bwd(P, P, 0, 4, 8, 8, 8, None, 0, stats["mean"], stats["rstd"], P, 8, None, None, None, 0,
                                     None) == ALIGNMENT


@pytest.mark.parametrize("a,b", [(ODD, P), (P, ODD)])
def test_product_factors(a, b):
    assert N.load().f8b200_gemm_blockwise(P, 0, 0, 16, a, 1, 1, 1, None, P, 0, 0, 16, b, 1, 1, 128, None, None, 0, P, 4, 4, 4, 16,
                                          None, 0, None) == ALIGNMENT
