"""Block-scaled training layers in uses beside the usual one."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from float8_experimental_b200 import _native as N, CastConfig, clip_grad_norm_, Float8LinearConfig, LayerNorm, ScalingType
from float8_experimental_b200.float8_linear import Float8Linear

pytestmark = pytest.mark.gpu

BF, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    torch.cuda.synchronize()
    assert N.read_device_error() == 0


def layer_of(k, n, dtype=BF, bias=True):
    torch.manual_seed(0)
    c = CastConfig(scaling_type=ScalingType.BLOCKWISE)
    config = Float8LinearConfig(cast_config_input=c, cast_config_weight=c, cast_config_grad_output=c)
    return Float8Linear.from_float(torch.nn.Linear(k, n, bias=bias, device="cuda", dtype=dtype), config)


@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("kind", ["strided", "expanded", "column", "fp32 strided"])
def test_bias_of_any_layout(m, kind):
    layer = layer_of(256, 192)
    buf = torch.randn(192 * 4, device="cuda")
    dense = {"strided": buf[: 2 * 192 : 2], "fp32 strided": buf[: 2 * 192 : 2], "expanded": buf[5:6].expand(192),
             "column": buf.view(192, 4)[:, 2]}[kind]
    if not kind.startswith("fp32"):
        wide = buf.to(BF)
        view = {"strided": wide[: 2 * 192 : 2], "expanded": wide[5:6].expand(192), "column": wide.view(192, 4)[:, 2]}[kind]
    else:
        view = dense
    x = torch.randn(m, 256, device="cuda").to(BF)
    layer.bias = torch.nn.Parameter(view.contiguous())
    want = layer(x)
    layer.bias = torch.nn.Parameter(view)
    assert layer.bias.stride() == view.stride() != (1,)
    y = layer(x)
    assert torch.equal(y, want)
    y.sum().backward()
    assert torch.equal(layer.bias.grad, torch.full((192,), float(m), device="cuda").to(view.dtype))


def test_bias_of_another_length_is_refused():
    layer = layer_of(256, 192)
    for length in (10, 193):
        layer.bias = torch.nn.Parameter(torch.zeros(length, device="cuda", dtype=BF))
        with pytest.raises(RuntimeError, match="the bias must have 192 elements"):
            layer(torch.zeros(4, 256, device="cuda", dtype=BF))


def test_captured_training_step():
    """Norm, layer, backward and clipping captured once and replayed on other inputs: the eager step's bits."""
    model = torch.nn.Sequential(LayerNorm(512, device="cuda", dtype=BF), layer_of(512, 384))
    params = list(model.parameters())
    x = torch.randn(300, 512, device="cuda").to(BF).requires_grad_()
    go = (torch.randn(300, 384, device="cuda") * 1e-2).to(BF)

    def step():
        for t in (x, *params):
            t.grad = None
        y = model(x)
        y.backward(go)
        return y, clip_grad_norm_(params, 1e-2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, total = step()
    with torch.no_grad():
        x.copy_(torch.randn(300, 512, device="cuda") * 3)
        go.copy_(torch.randn(300, 384, device="cuda") * 1e-3)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.detach().clone() for t in (y, total, x.grad, *(p.grad for p in params))]
    y2, total2 = step()
    assert all(torch.equal(a, b) for a, b in zip(got, (y2, total2, x.grad, *(p.grad for p in params))))


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_forward(reentrant):
    layer = layer_of(256, 192)
    x = torch.randn(200, 256, device="cuda").to(BF).requires_grad_()
    go = torch.randn(200, 192, device="cuda").to(BF)
    layer(x).backward(go)
    want = [t.grad for t in (x, layer.weight, layer.bias)]
    for t in (x, layer.weight, layer.bias):
        t.grad = None
    checkpoint(layer, x, use_reentrant=reentrant).backward(go)
    assert all(torch.equal(t.grad, w) for t, w in zip((x, layer.weight, layer.bias), want))


def test_two_backward_passes_of_one_forward():
    layer = layer_of(256, 192)
    x = torch.randn(200, 256, device="cuda").to(BF).requires_grad_()
    gos = [torch.randn(200, 192, device="cuda").to(BF) for _ in range(2)]
    y = layer(x)
    got = [torch.autograd.grad(y, [x, layer.weight], go, retain_graph=True) for go in gos]
    with torch.no_grad():
        layer.weight.add_(1)  # an optimiser's step in between: the graph holds the weight's cast
    again = [torch.autograd.grad(y, [x, layer.weight], go, retain_graph=True) for go in gos]
    for a, b in zip(got, again):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_compiled_training_step():
    """The traced forward and backward run the same kernels."""
    torch._dynamo.reset()
    layer = layer_of(256, 192)
    x = torch.randn(200, 256, device="cuda").to(BF).requires_grad_()
    go = torch.randn(200, 192, device="cuda").to(BF)
    leaves = [x, layer.weight, layer.bias]
    want = [layer(x), *torch.autograd.grad(layer(x), leaves, go)]
    y = torch.compile(layer, backend="aot_eager")(x)
    got = [y, *torch.autograd.grad(y, leaves, go)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
