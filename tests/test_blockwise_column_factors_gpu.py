"""Products with a factor per row on both sides whose CTA pairs take several tiles of an odd number of k-blocks: the
column factors of one tile's last block and the next tile's first must not share a buffer."""
import pytest
import torch

from blockwise_reference import product, product_tolerance
from float8_experimental_b200 import _native as N
from float8_experimental_b200._ops import ops

pytestmark = pytest.mark.gpu

E4, FP32 = torch.float8_e4m3fn, torch.float32


@pytest.mark.parametrize("k", [128, 384, 640])
@pytest.mark.parametrize("m,n", [(1000, 8192), (2300, 4100)])
def test_several_tiles_of_odd_depth(m, n, k):
    gen = torch.Generator(device="cuda").manual_seed(k)
    a, b = ((torch.randn(rows, k, device="cuda", generator=gen) * 60).to(E4) for rows in (m, n))
    # neighbouring rows of B differ by powers of ten: another tile's factors would show
    sa = torch.rand(m, k // 128, device="cuda", generator=gen) + 0.1
    sb = 10.0 ** torch.randint(-4, 5, (n, k // 128), device="cuda", generator=gen)
    first = ops.blockwise_mm(a, b, sa, sb, 1, 1, None, None, None, FP32)
    ref, mag = product(a, sa, 1, b, sb, 1)
    assert float(((first.double() - ref).abs() - product_tolerance(ref, mag, k, FP32)).max()) <= 0
    for _ in range(20):
        assert torch.equal(first, ops.blockwise_mm(a, b, sa, sb, 1, 1, None, None, None, FP32))
    assert N.read_device_error() == 0
