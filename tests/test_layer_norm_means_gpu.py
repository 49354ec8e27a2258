"""Rows whose mean is large against their spread, at widths whose reciprocal is no fp32 number."""
import pytest
import torch

from blockwise_reference import layer_norm as reference
from float8_experimental_b200.layer_norm import layer_norm

pytestmark = pytest.mark.gpu

BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24  # half a step of fp32
WIDTHS = [96, 1000, 1030, 7168, 20001]


def depth(cols):
    """Additions one value goes through in a sum over a row: 256 threads (32 in narrow rows), then the tree."""
    return cols / 32 + 16 if cols <= 1024 else cols / 256 + 16


def errors(x, eps):
    """(off, rel): how far n * std may be off, and the relative error of rstd.  The first mean m is off by
    e = (d + 2) U mean|x|; its rest r is a sum of x - m, off by d U of their mean size and three roundings; the variance's
    relative error is d U of sum(x - m)^2 = C (var + e^2), and the roundings of its terms."""
    xd = x.double()
    d = depth(x.shape[-1])
    mean = xd.mean(-1, keepdim=True)
    var = (xd - mean).square().mean(-1, keepdim=True)
    e = (d + 2) * U * xd.abs().mean(-1, keepdim=True)
    size = (xd - mean).abs().mean(-1, keepdim=True) + e
    off = (d + 4) * U * size + 2 * U * ((xd - mean).abs() + e)
    rel = (d + 8) * U * (var + e * e + eps) / (var + eps)
    return off, rel


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("spread", [1e-2, 1.0])
@pytest.mark.parametrize("affine", [False, True])
def test_large_means(cols, spread, affine):
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x = 1000.0 + spread * torch.randn(24, cols, device="cuda", generator=gen)
    w = 1 + 0.2 * torch.randn(cols, device="cuda", generator=gen) if affine else None
    b = 0.3 * torch.randn(cols, device="cuda", generator=gen) if affine else None
    eps = 1e-9
    y = layer_norm(x, w, b, eps)
    ref, n, rstd, _ = reference(x, w, b, eps)
    off, rel = errors(x, eps)
    size = 1.0 if w is None else w.double().abs()
    tol = size * (rstd * off + n.abs() * rel) + 3 * U * (ref.abs() + size * n.abs())
    assert float(((y.double() - ref).abs() - tol).max()) <= 0


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("eps", [1e-5, 1e-12])
def test_constant_rows(cols, dtype, eps):
    """Every element is the mean: what is left is the rounding of the rest, times at most 1 / sqrt(eps)."""
    x = torch.tensor([1000.0, -7.25, 0.0, 3.0, 1e-3], device="cuda").to(dtype)[:, None].expand(5, cols).contiguous()
    y = layer_norm(x, eps=eps)
    off, _ = errors(x, eps)
    assert bool((y.double().abs() <= off * eps ** -0.5 * (1 + 1e-5)).all())


@pytest.mark.parametrize("cols", WIDTHS)
def test_gradients_with_large_means(cols):
    """The backward pass's n takes the stored mean, which fp32 rounds by half a step of it."""
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x = (1000.0 + torch.randn(24, cols, device="cuda", generator=gen)).requires_grad_()
    w = (1 + 0.2 * torch.randn(cols, device="cuda", generator=gen)).requires_grad_()
    g = torch.randn(24, cols, device="cuda", generator=gen)
    eps = 1e-5
    dx, dw = torch.autograd.grad(layer_norm(x, w, eps=eps), [x, w], g)
    xd, wd, gd = x.detach().double(), w.detach().double(), g.double()
    _, n, rstd, mean = reference(xd, wd, None, eps)
    off, rel = errors(x.detach(), eps)
    d = depth(cols)
    e_n = rstd * (off + U * (mean.abs() + 2)) + n.abs() * (rel + 4 * U)
    h = gd * wd
    hn = (h * n).abs().mean(-1, keepdim=True)
    ref = rstd * (h - h.mean(-1, keepdim=True) - n * (h * n).mean(-1, keepdim=True))
    tol = rstd * ((d + 8) * U * (h.abs() + h.abs().mean(-1, keepdim=True) + n.abs() * hn) + e_n * hn +
                  n.abs() * (h.abs() * e_n).mean(-1, keepdim=True)) + ref.abs() * (rel + 8 * U)
    assert float(((dx.double() - ref).abs() - tol).max()) <= 0
    tol = (24 + 8) * U * (gd * n).abs().sum(0) + (gd.abs() * e_n).sum(0)
    assert float(((dw.double() - (gd * n).sum(0)).abs() - tol).max()) <= 0


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype", [BF, FP32])
def test_squares_that_overflow(cols, dtype):
    """The variance is infinite, so every value is zero deviations from the mean; other rows are as they are alone."""
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(6, cols, device="cuda", generator=gen).to(dtype)
    alone = layer_norm(x)
    x[1] = 1e30
    x[3] *= 1e25
    x[4] = x[4] * 1e25 + 1e30
    y = layer_norm(x)
    assert bool((y[[1, 3, 4]] == 0).all())
    assert torch.equal(y[[0, 2, 5]], alone[[0, 2, 5]])
