"""The shape functions that traces see against the implementations (their launches left out): sizes, strides, types and
which results share memory."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from float8_experimental_b200 import _native as N, _ops
from float8_experimental_b200._ops import ops

BF, E4, FP32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32


@pytest.fixture(autouse=True)
def no_launches(monkeypatch):
    for name in ("cast_blockwise", "uncast_blockwise", "gemm_blockwise", "layer_norm", "layer_norm_bwd", "multi_norm"):
        monkeypatch.setattr(N, name, lambda *a, **k: None)
    monkeypatch.setattr(_ops, "TensorList", lambda what, xs: xs)


def q(rows, cols):
    return torch.zeros(rows, cols).to(E4)


def stats(n):
    return torch.zeros(n), torch.zeros(n)


X = torch.zeros(130, 264, dtype=BF)
CASES = {
    "cast both": (ops.cast_blockwise, _ops._cast_blockwise_cuda, (X, 0, True, True)),
    "cast rows": (ops.cast_blockwise, _ops._cast_blockwise_cuda, (X[:, :33], 0, True, False)),
    "cast columns": (ops.cast_blockwise, _ops._cast_blockwise_cuda, (X.t(), 1, False, True)),
    "cast nothing": (ops.cast_blockwise, _ops._cast_blockwise_cuda, (X[:0], 0, True, True)),
    "square": (ops.cast_blockwise_square, _ops._cast_blockwise_square_cuda, (X, 0)),
    "square odd": (ops.cast_blockwise_square, _ops._cast_blockwise_square_cuda, (X[:7, :5], 1)),
    "uncast": (ops.uncast_blockwise, _ops._uncast_blockwise_cuda, (q(256, 384), torch.ones(256, 3), 1, 128, BF)),
    "uncast transposed": (ops.uncast_blockwise, _ops._uncast_blockwise_cuda,
                          (q(256, 384).t(), torch.ones(256, 3).t(), 128, 1, FP32)),
    "uncast transposed slice": (ops.uncast_blockwise, _ops._uncast_blockwise_cuda,
                                (q(256, 400)[:, :300].t(), torch.ones(3, 2), 128, 128, BF)),
    "uncast one row": (ops.uncast_blockwise, _ops._uncast_blockwise_cuda, (q(256, 1).t(), torch.ones(1, 2), 1, 128, BF)),
    "uncast one column": (ops.uncast_blockwise, _ops._uncast_blockwise_cuda, (q(1, 300).t(), torch.ones(300, 1), 1, 128, BF)),
    "uncast strided": (ops.uncast_blockwise, _ops._uncast_blockwise_cuda, (q(64, 256)[:, ::2], torch.ones(64, 1), 1, 128, BF)),
    "product": (ops.blockwise_mm, _ops._blockwise_mm_cuda,
                (q(130, 256), q(40, 256), torch.ones(130, 2), torch.ones(1, 2), 1, 128, None, None, torch.ones(40), torch.float16)),
    "layer norm": (ops.layer_norm, _ops._layer_norm_cuda, (X, None, None, 1e-5, True)),
    "layer norm strided": (ops.layer_norm, _ops._layer_norm_cuda, (torch.zeros(3, 8, 5).transpose(1, 2), None, None, 1e-5, True)),
    "layer norm alone": (ops.layer_norm, _ops._layer_norm_cuda, (X, None, None, 1e-5, False)),
    "layer norm backward": (ops.layer_norm_bwd, _ops._layer_norm_bwd_cuda, (X, X, None, *stats(130), FP32, True, True, True)),
    "layer norm backward, x": (ops.layer_norm_bwd, _ops._layer_norm_bwd_cuda,
                               (X.t(), X.t(), None, *stats(264), BF, True, False, False)),
    "layer norm backward, bias": (ops.layer_norm_bwd, _ops._layer_norm_bwd_cuda, (X, X, None, *stats(130), BF, False, False, True)),
    "norm": (ops.multi_norm, _ops._multi_norm_cuda, ([X, X[0]], 2, True)),
}


def described(out):
    outs = list(out) if isinstance(out, (tuple, list)) else [out]
    # a stride says nothing where a dimension has one element or the tensor none
    strides = [tuple(st for size, st in zip(t.shape, t.stride()) if size != 1) if t.numel() else () for t in outs]
    shared = [[t.untyped_storage()._cdata == u.untyped_storage()._cdata for u in outs] for t in outs]
    return [(tuple(t.shape), st, t.dtype, t.is_contiguous()) for t, st in zip(outs, strides)], shared


@pytest.mark.parametrize("name", CASES)
def test_fake_results_are_laid_out_like_real_ones(name):
    op, real, args = CASES[name]
    with FakeTensorMode() as mode:
        fake = op(*(mode.from_tensor(a) if isinstance(a, torch.Tensor) else
                    [mode.from_tensor(t) for t in a] if isinstance(a, list) else a for a in args))
    assert described(fake) == described(real(*args))
