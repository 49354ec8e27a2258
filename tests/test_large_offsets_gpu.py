"""Matrices and gradients of more than 2^31 elements: what lies behind that offset equals the same rows on their own."""
import gc

import pytest
import torch

from float8_experimental_b200 import _native as N, clip_grad_norm_, get_total_norm
from float8_experimental_b200._ops import ops
from float8_experimental_b200.float8_blockwise import blockwise_mm, cast_to_float8_blockwise, cast_to_float8_blockwise_both
from float8_experimental_b200.layer_norm import layer_norm

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
ROWS, COLS, TAIL = (1 << 18) + 384, 8192, 256  # 2^31 + 3 million elements; a multiple of 128 rows


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    torch.cuda.synchronize()
    assert N.read_device_error() == 0
    gc.collect()
    torch.cuda.empty_cache()


def large():
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(ROWS, COLS, dtype=BF, device="cuda")
    block = torch.randn(1 << 14, COLS, device="cuda", generator=gen).to(BF)
    for at in range(0, ROWS, 1 << 14):
        rows = min(1 << 14, ROWS - at)
        x[at:at + rows] = block[:rows]
    x[-TAIL:] = torch.randn(TAIL, COLS, device="cuda", generator=gen)
    return x


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_casts_and_products():
    x = large()
    tail = x[-TAIL:].clone()
    (r, c), (tr, tc) = cast_to_float8_blockwise_both(x), cast_to_float8_blockwise_both(tail)
    s, ts = cast_to_float8_blockwise(x, (128, 128)), cast_to_float8_blockwise(tail, (128, 128))
    w = cast_to_float8_blockwise(torch.randn(200, COLS, device="cuda").to(BF), (128, 128))
    # both by the tensor cores' factors: the same sums, tile for tile
    assert torch.equal(blockwise_mm(r, w.t())[-TAIL:], blockwise_mm(tr, w.t()))
    for a, b in ((r, tr), (c, tc), (s, ts)):
        assert same(a.data[-TAIL:], b.data)
        n = b.scale_inv.shape[0]
        assert torch.equal(a.scale_inv[-n:], b.scale_inv)
        assert torch.equal(a.to_original_precision()[-TAIL:], b.to_original_precision())
    assert torch.equal(ops.blockwise_mm(r.data, w.data, r.scale_inv, w.scale_inv, 1, 128, None, None, None, BF)[-TAIL:],
                       ops.blockwise_mm(tr.data, w.data, tr.scale_inv, w.scale_inv, 1, 128, None, None, None, BF))


def test_a_large_output():
    """More than 2^31 results, from few k."""
    a, b = (torch.randn(n, 128, device="cuda").to(BF) for n in (ROWS, COLS))
    a8, b8 = cast_to_float8_blockwise(a), cast_to_float8_blockwise(b, (128, 128))
    t8 = cast_to_float8_blockwise(a[-TAIL:].clone())
    assert torch.equal(blockwise_mm(a8, b8.t())[-TAIL:], blockwise_mm(t8, b8.t()))


def test_layer_norm_both_ways():
    x = large()
    tail = x[-TAIL:].clone()
    w, b = torch.randn(COLS, device="cuda").to(BF), torch.randn(COLS, device="cuda").to(BF)
    y, mean, rstd = ops.layer_norm(x, w, b, 1e-5, True)
    ty, tmean, trstd = ops.layer_norm(tail, w, b, 1e-5, True)
    assert torch.equal(y[-TAIL:], ty) and torch.equal(mean[-TAIL:], tmean) and torch.equal(rstd[-TAIL:], trstd)
    del y
    dx, _, _ = ops.layer_norm_bwd(x, x, w, mean, rstd, BF, True, True, True)
    tdx, _, _ = ops.layer_norm_bwd(tail, tail, w, tmean, trstd, BF, True, True, True)
    assert torch.equal(dx[-TAIL:], tdx)
    del dx
    odd = x.view(-1)[: (ROWS - 1) * COLS].view(-1, COLS)[:, : COLS - 1]  # rows that allow no wide accesses
    assert torch.equal(layer_norm(odd)[-100:], layer_norm(odd[-100:].clone()))


def test_one_large_gradient():
    g = large().view(-1)
    p = torch.nn.Parameter(torch.empty(0, device="cuda", dtype=BF))
    p.data = torch.empty_like(g)
    p.grad = g
    want = sum(float(part.double().square().sum()) for part in g.split(1 << 27)) ** 0.5
    before = g[-1000:].clone()
    assert abs(float(get_total_norm([g])) - want) <= 70 * 2.0 ** -24 * want
    assert abs(float(clip_grad_norm_([p], want / 2)) - want) <= 70 * 2.0 ** -24 * want
    assert torch.allclose(g[-1000:].float(), before.float() / 2, rtol=2.0 ** -7)
