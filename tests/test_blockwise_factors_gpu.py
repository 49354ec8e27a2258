"""Products follow the factors that a block tensor holds, however they came to be written."""
import pytest
import torch

from blockwise_reference import product, product_tolerance
from float8_experimental_b200 import _native as N
from float8_experimental_b200._ops import ops
from float8_experimental_b200.float8_blockwise import blockwise_mm, cast_to_float8_blockwise, cast_to_float8_blockwise_both

pytestmark = pytest.mark.gpu

BF, FP32 = torch.bfloat16, torch.float32
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def operands(m):
    gen = torch.Generator(device="cuda").manual_seed(m)
    return (torch.randn(rows, 512, device="cuda", generator=gen).to(BF) for rows in (m, 384))


WRITES = {"assigned": lambda t: setattr(t, "scale_inv", t.scale_inv * 3), "in place": lambda t: t.scale_inv.mul_(3),
          "data": lambda t: t.scale_inv.data.mul_(3), "half": lambda t: t.scale_inv[::2].mul_(3)}


@pytest.mark.parametrize("m", [20, 300])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("how", WRITES)
def test_written_factors_count(m, side, how):
    x, w = operands(m)
    a, b = cast_to_float8_blockwise(x), cast_to_float8_blockwise(w, (128, 128))
    before = b.t()  # shares b's factors
    WRITES[how]((a, b)[side])
    for second in (b.t(), before) if how != "assigned" else (b.t(),):
        got = blockwise_mm(a, second, FP32)
        ref, mag = product(a.data, a.scale_inv, 1, b.data, b.scale_inv, 128)
        assert float(((got - ref).abs() - product_tolerance(ref, mag, 512, FP32)).max()) <= 0
    assert N.read_device_error() == 0


@pytest.mark.parametrize("inference", [False, True])
def test_untouched_casts_go_to_the_tensor_cores_factors(inference):
    """The same bits as the product that is given the cast's exponent bytes."""
    x, w = operands(300)
    with torch.inference_mode(inference):
        got = blockwise_mm(cast_to_float8_blockwise(x), cast_to_float8_blockwise(w, (128, 128)).t(), FP32)
    x8, sx, ex = ops.cast_blockwise(x, N.E4M3, True, False)[:3]
    w8, sw, ew, _ = ops.cast_blockwise_square(w, N.E4M3)
    # other factors beside the same exponent bytes: only the kernel that reads the bytes gives the same result
    want = ops.blockwise_mm(x8, w8, torch.zeros_like(sx), torch.zeros_like(sw), 1, 128, ex, ew, None, FP32)
    assert torch.equal(got, want) and float(got.abs().max()) > 0


@pytest.mark.parametrize("m,n,k", [(129, 128, 128), (200, 256, 512), (300, 260, 640), (513, 1000, 1030), (140, 77, 2333),
                                   (4100, 600, 520)])
@pytest.mark.parametrize("out", [BF, torch.float16, FP32])
@pytest.mark.parametrize("kinds", [(E4, E4), (E4, E5), (E5, E4)])
def test_products_of_untouched_casts(m, n, k, out, kinds):
    """All three products of a layer, their factors applied by the tensor cores, against the doubles of what the casts stand for;
    a NaN poisons what its blocks reach."""
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    x = torch.randn(m, k, device="cuda", generator=gen) * torch.exp2(torch.randint(-12, 8, (m, k), device="cuda", generator=gen))
    x[m // 2], x[m // 3], x[0, : k // 2] = 0.0, 1e3, 1e-30
    x[17, 3] = float("nan")
    w, g = (torch.randn(*s, device="cuda", generator=gen).to(BF) for s in ((n, k), (m, n)))
    (xr, xc), (gr, gc) = (cast_to_float8_blockwise_both(t.to(BF), kinds[0]) for t in (x, g))
    w8 = cast_to_float8_blockwise(w, (128, 128), kinds[1])
    b = torch.randn(n, device="cuda", generator=gen).to(out)
    cases = [(xr, w8, b, k), (gr, w8.t(), None, n), (gc.t(), xc.t(), None, m)]
    results = [blockwise_mm(a, bt.t(), out, bias) for a, bt, bias, _ in cases]
    for got, (a, bt, bias, kk) in zip(results, cases):
        ref, mag = product(a.data, a.scale_inv, a.block[0], bt.data, bt.scale_inv, bt.block[0], bias)
        err = (got.double() - ref).abs() - product_tolerance(ref, mag, kk, out)
        fits = ref.abs() < torch.finfo(out).max * 0.99
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert float(torch.where(fits, err, -1.0).max()) <= 0
    assert N.read_device_error() == 0
