"""Block-scaled training layers in uses beside the usual one."""
import pytest
import torch

from float8_experimental_b200 import _native as N, CastConfig, Float8LinearConfig, ScalingType
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
