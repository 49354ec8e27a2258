"""Calls under traces and dispatch modes: the operators are seen, and a replay computes them."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from float8_experimental_b200 import CastConfig, clip_grad_norm_, Float8LinearConfig, get_total_norm, ScalingType
from float8_experimental_b200.float8_blockwise import blockwise_mm, cast_to_float8_blockwise, cast_to_float8_blockwise_both
from float8_experimental_b200.float8_linear import Float8Linear
from float8_experimental_b200.inference import ActivationCasting, quantize_to_float8, QuantConfig
from float8_experimental_b200.layer_norm import layer_norm

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "f8b200":
            self.names.append(func.__name__.split(".")[0])
        return func(*args, **(kwargs or {}))


def blockwise_layer(k=256, n=192):
    torch.manual_seed(0)
    c = CastConfig(scaling_type=ScalingType.BLOCKWISE)
    return Float8Linear.from_float(torch.nn.Linear(k, n, device="cuda", dtype=BF),
                                   Float8LinearConfig(cast_config_input=c, cast_config_weight=c, cast_config_grad_output=c))


def inference_layer():
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(256, 192, device="cuda", dtype=BF))
    quantize_to_float8(model, QuantConfig(ActivationCasting.BLOCKWISE))
    return model


def casts(x):
    a, b = cast_to_float8_blockwise_both(x)
    w = cast_to_float8_blockwise(x[:160], (128, 128))
    return blockwise_mm(a, w.t(), torch.float32), b.to_original_precision(), a.t().to_original_precision()


LAYER, INFERENCE = [], []  # without gradients: jit.trace takes what a function closes over as constants


def training(x):
    with torch.no_grad():
        return LAYER[0](x)


CALLS = {"casts and product": (casts, {"cast_blockwise", "cast_blockwise_square", "blockwise_mm", "uncast_blockwise"}),
         "layer norm": (lambda x: layer_norm(x, x[0], x[1]), {"layer_norm"}),
         "total norm": (lambda x: get_total_norm([x[:7], x[9:]]), {"multi_norm"}),
         "training layer": (training, {"cast_blockwise", "cast_blockwise_square", "blockwise_mm"}),
         "inference layer": (lambda x: INFERENCE[0](x), {"cast_blockwise", "blockwise_mm"})}


@pytest.fixture(autouse=True)
def layers():
    LAYER[:], INFERENCE[:] = [blockwise_layer().requires_grad_(False)], [inference_layer().requires_grad_(False)]
    yield
    LAYER.clear()
    INFERENCE.clear()


def values(out):
    return list(out) if isinstance(out, (tuple, list)) else [out]


def inputs():
    gen = torch.Generator(device="cuda").manual_seed(3)
    return [torch.randn(200, 256, device="cuda", generator=gen).to(BF) for _ in range(2)]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("how", ["make_fx", "make_fx pre-dispatch", "jit.trace"])
def test_traces_hold_the_operators(name, how):
    call, _ = CALLS[name]
    first, second = inputs()
    want = [values(call(x)) for x in (first, second)]
    if how == "jit.trace":
        traced = torch.jit.trace(call, (first,), check_trace=False)
    else:
        traced = make_fx(call, pre_dispatch=how != "make_fx")(first)
    for x, outs in zip((first, second), want):
        # large products may differ in their last places: with and without the casts' exponent bytes
        for got, ref in zip(values(traced(x)), outs):
            assert torch.allclose(got.float(), ref.float(), rtol=2.0 ** -7, atol=1e-3)
            assert got.stride() == ref.stride()


@pytest.mark.parametrize("name", CALLS)
def test_modes_see_the_operators(name):
    call, names = CALLS[name]
    x, _ = inputs()
    want = values(call(x))
    with Seen() as seen:
        got = values(call(x))
    assert names <= set(seen.names)
    assert all(torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-3) for a, b in zip(got, want))


def test_clipping_under_a_mode():
    g = torch.full((100,), 3.0, device="cuda")
    p = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    p.grad = g
    with Seen() as seen:
        total = clip_grad_norm_([p], 3.0)
    assert seen.names == ["multi_norm", "multi_clip_"]
    assert float(total) == 30.0 and bool(((g - 0.3).abs() < 1e-6).all())


def test_watched_backward_of_an_eager_forward():
    layer = blockwise_layer()
    x, go = inputs()
    x.requires_grad_()
    go = go[:, :192].contiguous()
    leaves = [x, layer.weight, layer.bias]
    want = torch.autograd.grad(layer(x), leaves, go)
    y = layer(x)
    with Seen() as seen:
        got = torch.autograd.grad(y, leaves, go)
    assert seen.names.count("cast_blockwise") == 1 and seen.names.count("blockwise_mm") == 2
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    norm = layer_norm(x, layer.weight[0])
    with Seen() as seen:
        torch.autograd.grad(norm, [x], torch.ones_like(norm))
    assert seen.names == ["layer_norm_bwd"]
    # without the weight's gradient the by-column form was never made
    layer.weight.requires_grad_(False)
    y = layer(x)
    with Seen():
        dx, = torch.autograd.grad(y, [x], go)
    assert torch.equal(dx, want[0])


@pytest.mark.parametrize("name", CALLS)
def test_compiled(name):
    call, _ = CALLS[name]
    first, second = inputs()
    want = [values(call(x)) for x in (first, second)]
    compiled = torch.compile(call, backend="aot_eager", fullgraph=name in ("layer norm", "total norm"))
    for x, outs in zip((first, second), want):
        for got, ref in zip(values(compiled(x)), outs):
            assert torch.allclose(got.float(), ref.float(), rtol=2.0 ** -7, atol=1e-3) and got.stride() == ref.stride()


def test_compiled_clipping():
    grads = [torch.full((50,), 3.0, device="cuda"), torch.full((50,), 3.0, device="cuda", dtype=BF)]
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    total = torch.compile(lambda: clip_grad_norm_(params, 3.0), backend="aot_eager")()
    assert float(total) == 30.0
    assert all(bool(((g.float() - 0.3).abs() < 1e-2).all()) for g in grads)
