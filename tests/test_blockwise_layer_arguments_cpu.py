"""What the eager training layer hands to its kernels, with the launches replaced: runs without a GPU."""
import types

import pytest
import torch

from float8_experimental_b200 import _native as N
from float8_experimental_b200.float8_blockwise import _float8_linear_blockwise

M, K, OUT = 6, 32, 64


@pytest.fixture
def products(monkeypatch):
    """The bias of every product that would be launched."""
    seen = []
    monkeypatch.setattr(N, "block_cast_into", lambda *a: None)
    monkeypatch.setattr(N, "block_gemm_into", lambda a, b, bias, *rest: seen.append(bias))
    return seen


def forward(bias, dtype=torch.bfloat16):
    x, weight = torch.zeros(M, K, dtype=dtype), torch.zeros(OUT, K, dtype=dtype)
    ctx = types.SimpleNamespace(save_for_backward=lambda *t: None)
    return _float8_linear_blockwise._forward_eager(ctx, x, x, weight, bias, True)


BUF = torch.arange(4 * OUT, dtype=torch.float32).to(torch.bfloat16)
BIASES = {"dense": BUF[:OUT], "strided": BUF[: 2 * OUT : 2], "expanded": BUF[3:4].expand(OUT),
          "column": BUF.view(OUT, 4)[:, 1], "other type": torch.arange(2 * OUT, dtype=torch.float32)[::2]}


@pytest.mark.parametrize("name", BIASES)
def test_a_bias_of_any_layout_arrives_dense(products, name):
    bias = BIASES[name]
    forward(bias)
    got, = products
    assert got.is_contiguous() and got.shape == (OUT,) and got.dtype == torch.bfloat16
    assert torch.equal(got, bias.to(torch.bfloat16))


@pytest.mark.parametrize("shape", [(10,), (OUT + 1,), (1, OUT), (0,)])
def test_a_bias_of_another_length_is_refused(products, shape):
    with pytest.raises(RuntimeError, match=f"the bias must have {OUT} elements"):
        forward(torch.zeros(shape, dtype=torch.bfloat16))
    assert not products


def test_no_bias(products):
    forward(None)
    assert products == [None]
