"""Block-scaled casts and products on the GPU against 64-bit restatements."""
import gc
import pytest
import torch

import float8_experimental_b200 as f8
from blockwise_reference import cast as ref_cast, product, product_tolerance, spread
from float8_experimental_b200 import _native as N, CastConfig, Float8LinearConfig, ScalingType
from float8_experimental_b200._ops import ops
from float8_experimental_b200.float8_blockwise import (
    blockwise_mm, cast_to_float8_blockwise, cast_to_float8_blockwise_both, Float8BlockTensor,
)
from float8_experimental_b200.float8_linear import Float8Linear

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def leave_no_tensors():
    """What failed calls left in reference cycles (tracebacks hold their frames) goes now, not in the middle of another
    file's count of allocated bytes."""
    yield
    gc.collect()


E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    torch.cuda.synchronize()
    assert N.read_device_error() == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def wide(rows, cols, dtype, seed):
    """Values over many powers of two, some blocks zero, some tiny, some at the type's maximum."""
    x = randn(rows, cols, seed=seed) * torch.exp2(torch.randint(-12, 8, (rows, cols), device="cuda", generator=gen(seed + 1)))
    x = x.to(dtype)
    if rows > 2:
        x[rows // 2] = 0.0
        x[rows // 3] = torch.finfo(dtype).max
        x[0, : cols // 2] = torch.finfo(dtype).smallest_normal
    return x


def same(t, ref):
    """Equal values, NaN in the same places."""
    t = t.double()
    return bool(((t == ref) | (torch.isnan(t) & torch.isnan(ref))).all())


# ---- casts: every byte and factor equals the definition -----------------------------------------------
@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("fmt", [E4, E5])
@pytest.mark.parametrize("shape", [(1, 128), (128, 128), (1, 1), (3, 40), (130, 264), (257, 133), (64, 1000)])
def test_casts_equal_the_definition(dtype, fmt, shape):
    x = wide(*shape, dtype, seed=shape[0] + shape[1])
    forms = {(1, 128): cast_to_float8_blockwise(x, (1, 128), fmt), (128, 1): cast_to_float8_blockwise(x, (128, 1), fmt),
             (128, 128): cast_to_float8_blockwise(x, (128, 128), fmt)}
    both = cast_to_float8_blockwise_both(x, fmt)
    for block, t in forms.items():
        q, s = ref_cast(x, block, fmt)
        assert t.block == block and t.orig_dtype is dtype
        assert same(t.data, q), block
        assert same(t.scale_inv, s), block
        back = t.to_original_precision(FP32)
        assert same(back, (q.float() * spread(s.float(), block, x.shape)).double()), block
        assert same(t.t().to_original_precision(FP32).t(), back.double())
    for t, block in zip(both, ((1, 128), (128, 1))):
        assert torch.equal(t.data.view(torch.uint8), forms[block].data.view(torch.uint8))
        assert torch.equal(t.scale_inv, forms[block].scale_inv)


@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
def test_cast_every_16_bit_fraction(dtype):
    """Ties included: a bf16 or fp16 block holds every fraction once, next to each possible amax fraction."""
    base = torch.arange(0, 65536, dtype=torch.int32, device="cuda").to(torch.int16)
    vals = base.view(torch.float16 if dtype == FP16 else BF)
    vals = vals[torch.isfinite(vals)].to(dtype)
    vals = vals[: vals.numel() // 128 * 128].view(-1, 128)
    vals = vals[torch.randperm(vals.shape[0], device="cuda", generator=gen(1))[:200]]
    for block in ((1, 128), (128, 1), (128, 128)):
        t = cast_to_float8_blockwise(vals, block)
        q, s = ref_cast(vals, block, E4)
        assert same(t.data, q) and same(t.scale_inv, s)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
def test_nonfinite_values_poison_their_block_only(bad, dtype):
    x = randn(200, 300, seed=3).to(dtype)
    x[5, 7] = bad
    x[199, 299] = bad
    for block in ((1, 128), (128, 1), (128, 128)):
        t = cast_to_float8_blockwise(x, block)
        q, s = ref_cast(x, block, E4)
        assert same(t.data, q) and same(t.scale_inv, s)


def test_cast_of_strided_and_misaligned_inputs():
    big = randn(300, 520, seed=4).to(BF)
    for x in (big[:, :264], big[::2, 8:272], big[1:200, 3:100], big.t(), big[:0], big[:, :0]):
        a, b = cast_to_float8_blockwise_both(x)
        c, d = cast_to_float8_blockwise_both(x.contiguous().clone())
        assert torch.equal(a.data.view(torch.uint8), c.data.view(torch.uint8)) and torch.equal(a.scale_inv, c.scale_inv)
        assert torch.equal(b.data.view(torch.uint8), d.data.view(torch.uint8)) and torch.equal(b.scale_inv, d.scale_inv)


# ---- products -----------------------------------------------------------------------------------------
def operand(rows, k, fmt, block, seed, col_major=False):
    """fp8 [rows, k] of arbitrary values with arbitrary fp32 factors, the k axis last."""
    x = randn(rows, k, seed=seed) * (60.0 if fmt is E4 else 3000.0)
    q = x.to(fmt)
    s = torch.rand(-(-rows // block), -(-k // 128), device="cuda", generator=gen(seed + 7)) * 0.05 + 1e-3
    if col_major:
        buf = torch.empty(k, (rows + 15) // 16 * 16, dtype=torch.uint8, device="cuda")[:, :rows]
        buf.copy_(q.view(torch.uint8).t())
        q = buf.view(fmt).t()
        s = s.t().contiguous().t()
    return q, s


def check_product(m, n, k, a_block=1, b_block=128, fa=E4, fb=E4, out=BF, bias=False, a_mn=False, b_mn=False, seed=0):
    a, sa = operand(m, k, fa, a_block, seed, a_mn)
    b, sb = operand(n, k, fb, b_block, seed + 100, b_mn)
    bv = randn(n, seed=seed + 5).to(out) if bias else None
    got = ops.blockwise_mm(a, b, sa, sb, a_block, b_block, None, None, bv, out)
    ref, mag = product(a, sa, a_block, b, sb, b_block, bv)
    err = (got.double() - ref).abs() - product_tolerance(ref, mag, k, out)
    assert got.shape == (m, n) and got.dtype == out
    assert float(err.max()) <= 0, (m, n, k, float(err.max()))


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 100, 128, 129, 300])
@pytest.mark.parametrize("nk", [(128, 128), (256, 1024), (1000, 400), (8, 16), (24, 2064)])
def test_product_sizes(m, nk):
    check_product(m, *nk, out=FP32, seed=m)


@pytest.mark.parametrize("m", [40, 520])
@pytest.mark.parametrize("blocks", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("kinds", [(E4, E4), (E4, E5), (E5, E4), (E5, E5)])
def test_product_block_shapes_and_formats(m, blocks, kinds):
    check_product(m, 400, 528, *blocks, *kinds, out=FP32, seed=2)


@pytest.mark.parametrize("out", [BF, FP16, FP32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m", [3, 100, 513])
def test_product_outputs(out, bias, m):
    check_product(m, 328, 384, out=out, bias=bias, seed=3)


@pytest.mark.parametrize("a_mn,b_mn", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("m,n,k", [(48, 272, 400), (300, 272, 400), (130, 1000, 1030), (1, 64, 300)])
def test_product_memory_orders(a_mn, b_mn, m, n, k):
    for blocks in ((1, 128), (1, 1)):
        check_product(m, n, k, *blocks, out=FP32, a_mn=a_mn, b_mn=b_mn, seed=4)


@pytest.mark.parametrize("m,n,k", [(70, 77, 333), (1, 1, 1), (129, 1, 129), (300, 131, 4100)])
def test_product_odd_sizes(m, n, k):
    for out in (BF, FP32):
        check_product(m, n, k, out=out, bias=True, seed=5)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 8192), (64, 2048, 28672), (2048, 2304, 2048), (1000, 8192, 640)])
def test_product_large(m, n, k):
    check_product(m, n, k, out=BF, seed=6)
    check_product(m, n, k, b_block=1, out=BF, seed=7)


def test_product_strided_and_broadcast_factors():
    a, sa = operand(200, 512, E4, 1, 1)
    b, sb = operand(300, 512, E4, 128, 2)
    wide_sa = torch.zeros(400, 8, device="cuda")
    wide_sa[::2, ::2] = sa
    one = torch.full((1, 1), 0.25, device="cuda")
    for s in (wide_sa[::2, ::2], sa.t().contiguous().t()):
        ref, mag = product(a, sa, 1, b, sb, 128)
        got = ops.blockwise_mm(a, b, s, sb, 1, 128, None, None, None, FP32)
        assert float(((got - ref).abs() - product_tolerance(ref, mag, 512, FP32)).max()) <= 0
    got = ops.blockwise_mm(a, b, one.expand(200, 4), sb, 1, 128, None, None, None, FP32)
    ref, mag = product(a, one.expand(200, 4), 1, b, sb, 128)
    assert float(((got - ref).abs() - product_tolerance(ref, mag, 512, FP32)).max()) <= 0


def test_product_factors_need_not_be_scaled_alike():
    """Factors from 2^-60 to 2^60 in one row of blocks: nothing but the largest blocks counts."""
    for m in (20, 200):
        a, sa = operand(m, 640, E4, 1, 8)
        b, sb = operand(256, 640, E4, 128, 9)
        sa = sa * torch.tensor([2.0 ** -60, 1.0, 2.0 ** 60, 2.0 ** -30, 2.0 ** 30], device="cuda")
        got = ops.blockwise_mm(a, b, sa, sb, 1, 128, None, None, None, FP32)
        ref, mag = product(a, sa, 1, b, sb, 128)
        assert float(((got - ref).abs() - product_tolerance(ref, mag, 640, FP32)).max()) <= 0


def test_product_of_a_poisoned_block():
    for m in (30, 300):
        x, w = randn(m, 300, seed=1).to(BF), randn(200, 300, seed=2).to(BF)
        x[7, 150] = float("nan")
        w[130, 290] = float("inf")
        y = blockwise_mm(cast_to_float8_blockwise(x), cast_to_float8_blockwise(w, (128, 128)).t())
        bad = torch.zeros(m, 200, dtype=torch.bool, device="cuda")
        bad[7] = True
        bad[:, 128:] = True
        assert torch.equal(torch.isnan(y), bad)


@pytest.mark.parametrize("m,n,k", [(129, 128, 128), (200, 256, 512), (300, 260, 640), (513, 1000, 1030), (1, 200, 300),
                                   (140, 77, 2333), (4100, 600, 520)])
@pytest.mark.parametrize("out", [BF, FP16, FP32])
@pytest.mark.parametrize("kinds", [(E4, E4), (E4, E5), (E5, E4)])
def test_products_of_casts(m, n, k, out, kinds):
    """Operands from the casts, whose power-of-two factors the tensor cores apply: all three products of a layer, against
    the doubles of what the casts stand for."""
    x = wide(m, k, BF, seed=m).clamp(-1e3, 1e3)
    w, g = randn(n, k, seed=n).to(BF), randn(m, n, seed=k).to(BF)
    if m > 20:
        x[17, 3] = float("nan")
    xr, xc = cast_to_float8_blockwise_both(x, kinds[0])
    gr, gc = cast_to_float8_blockwise_both(g, kinds[0])
    w8 = cast_to_float8_blockwise(w, (128, 128), kinds[1])
    b = randn(n, seed=1).to(out)
    for a, bt, bias, kk in ((xr, w8, b, k), (gr, w8.t(), None, n), (gc.t(), xc.t(), None, m)):
        ref, mag = product(a.data, a.scale_inv, a.block[0], bt.data, bt.scale_inv, bt.block[0], bias)
        got = blockwise_mm(a, bt.t(), out, bias)
        err = (got.double() - ref).abs() - product_tolerance(ref, mag, kk, out)
        top = torch.finfo(out).max
        fits = ref.abs() < top * 0.99
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert float(torch.where(fits, err, -1.0).max()) <= 0


def test_factors_written_after_the_cast_count():
    for m in (20, 300):
        x = cast_to_float8_blockwise(randn(m, 256, seed=1).to(BF))
        w = cast_to_float8_blockwise(randn(128, 256, seed=2).to(BF), (128, 128))
        blockwise_mm(x, w.t(), FP32)
        x.scale_inv.mul_(2)
        # another kernel's order of summation: both are held to the doubles, not to each other's bits
        ref, mag = product(x.data, x.scale_inv, 1, w.data, w.scale_inv, 128)
        assert float(((blockwise_mm(x, w.t(), FP32) - ref).abs() - product_tolerance(ref, mag, 256, FP32)).max()) <= 0


def test_product_empty():
    e = cast_to_float8_blockwise
    b = torch.randn(256, device="cuda", dtype=BF)
    w = e(randn(256, 384, seed=1).to(BF), (128, 128))
    assert blockwise_mm(e(torch.empty(0, 384, device="cuda", dtype=BF)), w.t()).shape == (0, 256)
    none = Float8BlockTensor(torch.empty(256, 0, device="cuda", dtype=E4), torch.empty(2, 0, device="cuda"), (128, 128))
    y = blockwise_mm(e(torch.empty(5, 0, device="cuda", dtype=BF)), none.t(), bias=b)
    assert torch.equal(y, b.expand(5, 256))
    assert float(blockwise_mm(e(torch.empty(5, 0, device="cuda", dtype=BF)), none.t()).abs().max()) == 0


def test_product_repeats_to_the_bit():
    for m in (33, 700):
        a, sa = operand(m, 4096, E4, 1, 1)
        b, sb = operand(1024, 4096, E4, 1, 2)
        first = ops.blockwise_mm(a, b, sa, sb, 1, 1, None, None, None, FP32)
        for _ in range(5):
            assert torch.equal(first, ops.blockwise_mm(a, b, sa, sb, 1, 1, None, None, None, FP32))


# ---- the layers ---------------------------------------------------------------------------------------
def blockwise_config():
    c = CastConfig(scaling_type=ScalingType.BLOCKWISE)
    return Float8LinearConfig(cast_config_input=c, cast_config_weight=c, cast_config_grad_output=c)


def value(x, block):
    q, s = ref_cast(x, block, E4)
    return q * spread(s, block, x.shape)


@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("lead,k,n,bias", [((1,), 64, 48, True), ((2, 150), 272, 400, True), ((300,), 100, 33, False)])
def test_linear_forward_and_gradients(dtype, lead, k, n, bias):
    torch.manual_seed(0)
    lin = torch.nn.Linear(k, n, bias=bias, device="cuda", dtype=dtype)
    layer = Float8Linear.from_float(lin, blockwise_config())
    x = randn(*lead, k, seed=1).to(dtype).requires_grad_()
    go = (randn(*lead, n, seed=2) * 1e-2).to(dtype)
    y = layer(x)
    y.backward(go)
    x2, g2, w = x.detach().reshape(-1, k), go.reshape(-1, n), layer.weight.detach()
    m = x2.shape[0]
    xr, wq, gr = value(x2, (1, 128)), value(w, (128, 128)), value(g2, (1, 128))
    xc, gc = value(x2, (128, 1)), value(g2, (128, 1))
    b = layer.bias.detach().double() if bias else 0.0
    cases = [(y, xr @ wq.t() + b, xr.abs() @ wq.abs().t() + (b.abs() if bias else 0.0), k),
             (x.grad, gr @ wq, gr.abs() @ wq.abs(), n), (layer.weight.grad, gc.t() @ xc, gc.abs().t() @ xc.abs(), m)]
    for got, ref, mag, kk in cases:
        got = got.detach().reshape(ref.shape).double()
        assert float(((got - ref).abs() - product_tolerance(ref, mag, kk, dtype)).max()) <= 0
    if bias:
        ref, mag = g2.double().sum(0), g2.double().abs().sum(0)
        tol = torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 1e-6) + m * 2.0 ** -23 * mag + 1e-30
        assert float(((layer.bias.grad.double() - ref).abs() - tol).max()) <= 0


def test_linear_fp32_weight_under_autocast():
    lin = torch.nn.Linear(256, 128, device="cuda")
    layer = Float8Linear.from_float(lin, blockwise_config())
    x = randn(64, 256, seed=1).requires_grad_()
    with torch.autocast("cuda", torch.bfloat16):
        y = layer(x)
    assert y.dtype == BF
    y.float().sum().backward()
    assert layer.weight.grad.dtype == FP32 and x.grad.dtype == FP32
    ref, mag = value(x.detach().to(BF), (1, 128)), value(layer.weight.detach(), (128, 128))
    out, size = ref @ mag.t() + layer.bias.detach().to(BF).double(), ref.abs() @ mag.abs().t() + layer.bias.detach().double().abs()
    assert float(((y.detach().double() - out).abs() - product_tolerance(out, size, 256, BF)).max()) <= 0


def test_linear_partial_gradients_and_no_grad():
    lin = torch.nn.Linear(256, 128, device="cuda", dtype=BF)
    layer = Float8Linear.from_float(lin, blockwise_config())
    x = randn(64, 256, seed=1).to(BF)
    full = layer(x)
    with torch.no_grad():
        assert torch.equal(layer(x), full)
    go = randn(64, 128, seed=2).to(BF)
    dw, = torch.autograd.grad(layer(x), [layer.weight], go)
    layer.weight.requires_grad_(False)
    xr = x.clone().requires_grad_()
    dx, = torch.autograd.grad(layer(xr), [xr], go)
    layer.weight.requires_grad_(True)
    dx2, dw2 = torch.autograd.grad(layer(xr), [xr, layer.weight], go)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    # a broadcast gradient, no rows at all
    dx3, = torch.autograd.grad(layer(xr), [xr], torch.ones(1, 128, device="cuda", dtype=BF).expand(64, 128))
    dx4, = torch.autograd.grad(layer(xr), [xr], torch.ones(64, 128, device="cuda", dtype=BF))
    assert torch.equal(dx3, dx4)
    e = torch.empty(0, 256, device="cuda", dtype=BF, requires_grad=True)
    ye = layer(e)
    de, dwe = torch.autograd.grad(ye, [e, layer.weight], torch.empty(0, 128, device="cuda", dtype=BF))
    assert ye.shape == (0, 128) and de.shape == (0, 256) and float(dwe.abs().max()) == 0


@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("lead", [(1,), (3, 7), (200,)])
def test_inference_linear(dtype, lead):
    from float8_experimental_b200.inference import ActivationCasting, quantize_to_float8, QuantConfig

    model = torch.nn.Sequential(torch.nn.Linear(320, 200, device="cuda", dtype=dtype))
    w, b = model[0].weight.detach().clone(), model[0].bias.detach().clone()
    quantize_to_float8(model, QuantConfig(ActivationCasting.BLOCKWISE))
    x = randn(*lead, 320, seed=1).to(dtype)
    y = model(x)
    xr, wq = value(x.reshape(-1, 320), (1, 128)), value(w, (128, 128))
    ref, mag = xr @ wq.t() + b.double(), xr.abs() @ wq.abs().t() + b.double().abs()
    got = y.detach().reshape(ref.shape).double()
    assert y.shape == (*lead, 200) and float(((got - ref).abs() - product_tolerance(ref, mag, 320, dtype)).max()) <= 0
    # its state: bytes and factors, loadable
    state = {k: v.clone() for k, v in model.state_dict().items()}
    assert set(state) == {"0.weight", "0.bias", "0.weight_scale_inv"}
    other = torch.nn.Sequential(torch.nn.Linear(320, 200, device="cuda", dtype=dtype))
    quantize_to_float8(other, QuantConfig(ActivationCasting.BLOCKWISE))
    other.load_state_dict(state)
    assert torch.equal(other(x), y)


# ---- streams, graphs ----------------------------------------------------------------------------------
def test_streams_and_graphs():
    lin = torch.nn.Linear(512, 768, device="cuda", dtype=BF)
    layer = Float8Linear.from_float(lin, blockwise_config())
    xs = [randn(m, 512, seed=m).to(BF) for m in (5, 600)]
    with torch.no_grad():
        want = [layer(x) for x in xs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [layer(x) for x in xs]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        static = [x.clone() for x in xs]
        graphs, outs = [], []
        for x in static:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(layer(x))
            graphs.append(g)
        for x in static:
            x.mul_(-1)
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for _ in range(3):  # two graphs at once
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, layer(x)) for o, x in zip(outs, static))


def test_inference_mode():
    x, w = randn(200, 256, seed=1).to(BF), randn(64, 256, seed=2).to(BF)
    layer = Float8Linear.from_float(torch.nn.Linear(256, 64, device="cuda", dtype=BF), blockwise_config())
    want = layer(x).detach()
    with torch.inference_mode():
        a, b = cast_to_float8_blockwise(x), cast_to_float8_blockwise(w, (128, 128))
        y = blockwise_mm(a, b.t(), FP32)
        assert torch.equal(layer(x), want)
    ref, mag = product(a.data, a.scale_inv, 1, b.data, b.scale_inv, 128)
    assert float(((y - ref).abs() - product_tolerance(ref, mag, 256, FP32)).max()) <= 0


def test_saved_tensors_may_move():
    """A step whose saved tensors are packed away and come back as copies gives the same gradients."""
    layer = Float8Linear.from_float(torch.nn.Linear(384, 256, device="cuda", dtype=BF), blockwise_config())
    x, go = randn(300, 384, seed=1).to(BF).requires_grad_(), randn(300, 256, seed=2).to(BF)
    want = torch.autograd.grad(layer(x), [x, layer.weight, layer.bias], go)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        y = layer(x)
    got = torch.autograd.grad(y, [x, layer.weight, layer.bias], go)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals_on_the_gpu():
    a = cast_to_float8_blockwise(randn(8, 256, seed=1).to(BF))
    w = cast_to_float8_blockwise(randn(64, 256, seed=2).to(BF), (128, 128))
    with pytest.raises(ValueError, match="inner dimensions"):
        blockwise_mm(a, w)
    with pytest.raises(ValueError, match="128 long in the inner dimension"):
        blockwise_mm(cast_to_float8_blockwise(randn(8, 256, seed=1).to(BF), (128, 1)), w.t())
    with pytest.raises(RuntimeError, match="bias must have"):
        blockwise_mm(a, w.t(), bias=torch.zeros(63, device="cuda"))
    with pytest.raises(RuntimeError, match="scale_a must be"):
        ops.blockwise_mm(a.data, w.data, a.scale_inv[:, :1], w.scale_inv, 1, 128, None, None, None, BF)
    with pytest.raises(RuntimeError, match="different devices"):
        ops.blockwise_mm(a.data, w.data, a.scale_inv, w.scale_inv, 1, 128, None, None, torch.zeros(64), BF)
    with pytest.raises(N.F8B200Error, match="unsupported high-precision"):
        cast_to_float8_blockwise(torch.zeros(4, 4, device="cuda", dtype=torch.float64))
    layer = Float8Linear.from_float(torch.nn.Linear(256, 64, device="cuda", dtype=BF), blockwise_config())
    with pytest.raises(RuntimeError, match="plain tensors"):
        layer(f8.float8_tensor.hp_tensor_and_scale_to_float8(randn(8, 256).to(BF), torch.ones((), device="cuda")))
