"""Products of casts over a long inner dimension: the sums are fp32's however many blocks they run over."""
import pytest
import torch

from blockwise_reference import product
from float8_experimental_b200 import _native as N
from float8_experimental_b200.float8_blockwise import blockwise_mm, cast_to_float8_blockwise, cast_to_float8_blockwise_both

pytestmark = pytest.mark.gpu

BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def tolerance(ref, mag, k, out):
    """Half a step of the result's type.  A chunk of at most 2048 k (fp32 results; 4096 for 16-bit ones) is summed by the
    tensor cores in steps of 32, each off by at most one place of fp32 (2^-23 of the terms' magnitudes), the chunks
    and the bias are added with half a place each; 8 places for the sums inside the steps."""
    steps = 64 if out is FP32 else 128
    f = torch.finfo(out)
    return f.eps / 2 * ref.abs() * (1 + 1e-6) + (steps + 8 + k / (64 * steps)) * 2.0 ** -23 * mag + f.smallest_normal * f.eps


@pytest.mark.parametrize("out", [FP32, FP16, BF])
@pytest.mark.parametrize("k", [2048, 2049, 4224, 16384, 28700, 65536])
@pytest.mark.parametrize("signed", [False, True])
def test_long_sums(out, k, signed):
    gen = torch.Generator(device="cuda").manual_seed(k)
    x, w = (torch.randn(rows, k, device="cuda", generator=gen).mul_(0.8) for rows in (300, 260))
    if not signed:  # every step's error has the sign of the sum
        x, w = x.abs(), w.abs()
    a, b = cast_to_float8_blockwise(x.to(BF)), cast_to_float8_blockwise(w.to(BF), (128, 128))
    bias = torch.randn(260, device="cuda", generator=gen).to(out)
    got = blockwise_mm(a, b.t(), out, bias)
    ref, mag = product(a.data, a.scale_inv, 1, b.data, b.scale_inv, 128, bias)
    assert float(((got.double() - ref).abs() - tolerance(ref, mag, k, out)).max()) <= 0
    assert N.read_device_error() == 0


@pytest.mark.parametrize("out", [FP32, BF])
def test_long_sums_over_rows(out):
    """The weight gradient's form: both operands by columns, summed over many rows, several tiles per CTA pair."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens, n, k = 20000, 2560, 2304
    g, x = (torch.rand(tokens, cols, device="cuda", generator=gen).to(BF) for cols in (n, k))
    gc, xc = cast_to_float8_blockwise_both(g)[1], cast_to_float8_blockwise_both(x)[1]
    got = blockwise_mm(gc.t(), xc, out)
    again = blockwise_mm(gc.t(), xc, out)
    assert torch.equal(got, again)
    rows = torch.randint(0, n, (64,), device="cuda", generator=gen)
    ref, mag = product(gc.data.t()[rows], gc.scale_inv.t()[rows], 1, xc.data.t(), xc.scale_inv.t(), 1)
    assert float(((got[rows].double() - ref).abs() - tolerance(ref, mag, tokens, out)).max()) <= 0
    assert N.read_device_error() == 0
