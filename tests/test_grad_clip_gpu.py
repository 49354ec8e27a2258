"""Norm of many gradients and clipping, against 64-bit sums."""
import gc
import math

import pytest
import torch

from float8_experimental_b200 import clip_grad_norm_, clip_grads_with_norm_, get_total_norm
from float8_experimental_b200._ops import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def leave_no_tensors():
    """What failed calls left in reference cycles (tracebacks hold their frames) goes now, not in the middle of another
    file's count of allocated bytes."""
    yield
    gc.collect()


BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def params_of(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        out.append(p)
    return out


def exact_norm(grads, kind):
    flat = torch.cat([g.double().reshape(-1) for g in grads])
    return float(flat.abs().max() if kind == math.inf else flat.abs().sum() if kind == 1 else (flat * flat).sum().sqrt())


SIZES = {"one": [1], "small": [1, 2, 3, 7, 8, 9, 255, 256, 257, 0, 5], "chunks": [16384, 16383, 16385, 32768, 40000, 1],
         "many": [1 + (i * 37) % 900 for i in range(2500)], "large": [5_000_001, 3, 1 << 20]}


def make(sizes, dtype, seed):
    g = gen(seed)
    kinds = [BF, FP16, FP32] if dtype is None else [dtype]
    return [(torch.randn(s, device="cuda", generator=g) * 1e-2).to(kinds[i % len(kinds)]) for i, s in enumerate(sizes)]


@pytest.mark.parametrize("name", SIZES)
@pytest.mark.parametrize("dtype", [BF, FP16, FP32, None])
@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
def test_norm(name, dtype, kind):
    """64 squares per thread are added in fp32 (each addition half a step), all above it in fp64: 66 half steps of the
    sum, half of that in the root, and the final rounding.  The maximum is exact."""
    grads = make(SIZES[name], dtype, 1)
    got, want = get_total_norm(grads, kind), exact_norm(grads, kind)
    assert got.dtype == FP32 and got.dim() == 0
    assert abs(float(got) - want) <= (0.0 if kind == math.inf else 70 * 2.0 ** -24 * want)


@pytest.mark.parametrize("name", SIZES)
@pytest.mark.parametrize("dtype", [BF, FP16, FP32, None])
@pytest.mark.parametrize("share", [0.3, 3.0])
def test_clip(name, dtype, share):
    grads = make(SIZES[name], dtype, 2)
    before = [g.clone() for g in grads]
    norm = exact_norm(grads, 2.0)
    got = clip_grad_norm_(params_of(grads), share * norm)
    factor = min(1.0, share * norm / (norm + 1e-6))
    assert abs(float(got) - norm) <= 70 * 2.0 ** -24 * norm
    for g, old in zip(grads, before):
        if share > 1:
            assert torch.equal(g, old)
            continue
        want = old.double() * factor
        f = torch.finfo(g.dtype)
        # the norm's error, three roundings of the factor, one of the product, one to the type
        tol = want.abs() * (75 * 2.0 ** -24 + f.eps / 2 * (1 + 1e-6)) + f.smallest_normal * f.eps
        assert bool(((g.double() - want).abs() <= tol).all())


def test_misaligned_and_permuted_gradients():
    buf = torch.randn(100_000, device="cuda", generator=gen(3)).to(BF)
    views = [buf[1:5000], buf[5003:5003 + 20_000], buf[30_000:30_000 + 6000].view(60, 100).t(),
             buf[40_001:40_001 + 24_000].view(20, 30, 40).permute(2, 0, 1)]
    rest = buf.clone()
    want = [v.double() for v in views]
    norm = exact_norm([v.reshape(-1) for v in views], 2.0)
    for v in views:
        assert not v.is_contiguous() or v.data_ptr() % 16 != 0 or v.dim() == 1
    params = [torch.nn.Parameter(torch.empty_strided(v.shape, v.stride(), device="cuda", dtype=BF)) for v in views]
    for p, v in zip(params, views):
        p.grad = v
    clip_grad_norm_(params, 0.5 * norm)
    for v, w in zip(views, want):
        assert bool(((v.double() - 0.5 * w).abs() <= 0.5 * w.abs() * (2.0 ** -8 * 1.01) + 1e-7).all())
    # what lies between the gradients is as it was
    used = torch.zeros(100_000, dtype=torch.bool, device="cuda")
    for at, n in ((1, 4999), (5003, 20_000), (30_000, 6000), (40_001, 24_000)):
        used[at:at + n] = True
    assert torch.equal(buf[~used], rest[~used])


def test_nonfinite_norms():
    for bad in (float("nan"), float("inf")):
        for kind in (2.0, 1.0, math.inf):
            grads = [torch.ones(1000, device="cuda"), torch.ones(17, device="cuda", dtype=BF)]
            grads[1][3] = bad
            params = params_of(grads)
            with pytest.raises(RuntimeError, match="non-finite"):
                clip_grad_norm_(params, 1.0, kind, error_if_nonfinite=True)
            assert float(grads[0].min()) == 1.0
            total = clip_grad_norm_(params, 1.0, kind)
            assert math.isnan(float(total)) == math.isnan(bad) and not math.isfinite(float(total))
            if math.isnan(bad):
                assert bool(torch.isnan(grads[0]).all())
            else:
                assert float(grads[0].abs().max()) == 0.0 and math.isnan(float(grads[1][3]))


def test_zero_gradients_and_no_gradients():
    z = torch.zeros(100, device="cuda")
    assert float(clip_grad_norm_(params_of([z]), 1.0)) == 0.0 and float(z.abs().max()) == 0.0
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0
    assert float(get_total_norm([])) == 0.0
    e = torch.empty(0, device="cuda")
    assert float(get_total_norm([e])) == 0.0


def test_each_parameter_counts_once():
    g = torch.full((4,), 3.0, device="cuda")
    p, = params_of([g])
    assert float(clip_grad_norm_([p, p], 3.0)) == 6.0
    assert bool(((g - 1.5).abs() <= 1e-6).all())
    assert float(clip_grad_norm_(p, 100.0)) == pytest.approx(3.0, rel=1e-6)
    shared = torch.full((4,), 3.0, device="cuda")
    tied = params_of([shared, shared])
    assert float(clip_grad_norm_(tied, 3.0)) == 6.0
    assert bool(((shared - 1.5).abs() <= 1e-6).all())
    gen_params = (q for q in [p])
    assert float(clip_grad_norm_(gen_params, 100.0)) == pytest.approx(3.0, rel=1e-6)


def test_split_calls_streams_and_graphs():
    grads = make(SIZES["chunks"], None, 5)
    whole = [g.clone() for g in grads]
    clip_grad_norm_(params_of(whole), 0.01)
    params = params_of([g.clone() for g in grads])
    clip_grads_with_norm_(params, 0.01, get_total_norm([p.grad for p in params]))
    assert all(torch.equal(p.grad, w) for p, w in zip(params, whole))
    static = params_of([g.clone() for g in grads])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = clip_grad_norm_(static, 0.01)
    for p, g in zip(static, grads):
        p.grad.copy_(2 * g)
    graph.replay()
    torch.cuda.synchronize()
    twice = params_of([2 * g for g in grads])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = clip_grad_norm_(twice, 0.01)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(total, want) and all(torch.equal(a.grad, b.grad) for a, b in zip(static, twice))


def test_refusals_on_the_gpu():
    g = torch.zeros(4, 4, device="cuda")
    with pytest.raises(ValueError, match="norm_type"):
        get_total_norm([g], 3.0)
    with pytest.raises(RuntimeError, match="not dense"):
        get_total_norm([g[:, ::2]])
    with pytest.raises(RuntimeError, match="not dense"):
        get_total_norm([torch.zeros(1, device="cuda").expand(4)])
    with pytest.raises(RuntimeError, match="different devices"):
        get_total_norm([g, torch.zeros(4)])
    with pytest.raises(Exception, match="unsupported high-precision"):
        get_total_norm([g.double()])
    with pytest.raises(RuntimeError, match="one float32"):
        ops.multi_clip_([g], torch.zeros(2, device="cuda"), 1.0)


def test_norm_linear_clip_together():
    """A training step of the three, layer norm, block-scaled linear, backward, clipping: near the same step in 64 bits, and
    the same to the bit when it is repeated."""
    from float8_experimental_b200 import CastConfig, convert_to_float8_training, Float8LinearConfig, LayerNorm, ScalingType

    c = CastConfig(scaling_type=ScalingType.BLOCKWISE)
    config = Float8LinearConfig(cast_config_input=c, cast_config_weight=c, cast_config_grad_output=c)
    torch.manual_seed(0)
    model = torch.nn.Sequential(LayerNorm(256), torch.nn.Linear(256, 512), LayerNorm(512), torch.nn.Linear(512, 128)).cuda().to(BF)
    plain = [p.detach().clone() for p in model.parameters()]
    convert_to_float8_training(model, config=config)
    x = torch.randn(300, 256, device="cuda", generator=gen(1)).to(BF)
    go = torch.randn(300, 128, device="cuda", generator=gen(2)).to(BF) * 1e-2

    def step():
        for p in model.parameters():
            p.grad = None
        model(x).backward(go)
        return clip_grad_norm_(model.parameters(), 1e-3)

    total = step()
    grads = [p.grad for p in model.parameters()]
    # the same step in 64 bits without the casts to fp8
    w = [p.double().requires_grad_() for p in plain]
    ln = torch.nn.functional.layer_norm
    h = torch.nn.functional.linear(ln(x.double(), (256,), w[0], w[1]), w[2], w[3])
    y = torch.nn.functional.linear(ln(h, (512,), w[4], w[5]), w[6], w[7])
    ref = torch.autograd.grad(y, w, go.double())
    norm = math.sqrt(sum(float((r * r).sum()) for r in ref))
    # e4m3 rounds each factor of every product by up to 2^-4, 0.58 * 2^-4 on the average: signs differ, so the
    # gradients as a whole stay within twice that times the products' number along the way
    assert abs(float(total) - norm) <= 0.15 * norm
    clipped = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    assert abs(clipped - 1e-3) <= 1e-3 * 2.0 ** -8
    for g, r in zip(grads, ref):
        want = r * (1e-3 / norm)
        assert float((g.double() - want).norm()) <= 0.25 * float(want.norm())
    again = step()
    assert torch.equal(total, again)
    assert all(torch.equal(a, p.grad) for a, p in zip(grads, model.parameters()))
