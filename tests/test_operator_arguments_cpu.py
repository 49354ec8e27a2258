"""Arguments of the operators that are read by address: what does not fit is refused before a launch.  The launches are
replaced, so this runs without a GPU."""
import pytest
import torch

from float8_experimental_b200 import _native as N, _ops

BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def launches(monkeypatch):
    seen = []
    for name in ("layer_norm_bwd", "uncast_blockwise"):
        monkeypatch.setattr(N, name, lambda *a, name=name: seen.append(name))
    return seen


def backward(**changes):
    a = dict(x=torch.zeros(6, 8, dtype=BF), grad_y=torch.zeros(6, 8, dtype=BF), weight=torch.zeros(8, dtype=BF),
             mean=torch.zeros(6), rstd=torch.zeros(6), affine_dtype=BF, need_dx=True, need_dw=True, need_db=True)
    a.update(changes)
    return _ops._layer_norm_bwd_cuda(*a.values())


def test_layer_norm_backward_takes_what_fits(launches):
    backward()
    backward(weight=torch.zeros(8), affine_dtype=FP32)
    backward(weight=None)
    backward(weight=None, affine_dtype=FP32)
    backward(weight=torch.zeros(16, dtype=BF)[::2], grad_y=torch.zeros(1, 1, dtype=BF).expand(6, 8))
    backward(x=torch.zeros(2, 3, 8, dtype=BF), grad_y=torch.zeros(2, 3, 8, dtype=BF))
    assert len(launches) == 6


@pytest.mark.parametrize("changes,match", [
    (dict(grad_y=torch.zeros(6, 8)), "grad_y must be like x"),
    (dict(grad_y=torch.zeros(5, 8, dtype=BF)), "grad_y must be like x"),
    (dict(grad_y=torch.zeros(48, dtype=BF)), "grad_y must be like x"),
    (dict(mean=torch.zeros(5)), "mean must be 6"),
    (dict(rstd=torch.zeros(7)), "rstd must be 6"),
    (dict(mean=torch.zeros(6, dtype=BF)), "mean must be 6"),
    (dict(rstd=torch.zeros(12)[::2]), "rstd must be 6"),
    (dict(rstd=torch.zeros(1).expand(6)), "rstd must be 6"),
    (dict(mean=torch.zeros(6, 1)), "mean must be 6"),
    (dict(weight=torch.zeros(7, dtype=BF)), "one element per column"),
    (dict(weight=torch.zeros(8, dtype=FP16)), "both float32"),
    (dict(affine_dtype=FP32), "affine_dtype"),
    (dict(weight=torch.zeros(8)), "affine_dtype"),
    (dict(weight=None, affine_dtype=FP16), "affine_dtype"),
    (dict(x=torch.zeros(6, 0, dtype=BF), grad_y=torch.zeros(6, 0, dtype=BF)), "at least one element"),
])
def test_layer_norm_backward_refuses_what_does_not(launches, changes, match):
    with pytest.raises(RuntimeError, match=match):
        backward(**changes)
    assert not launches


Q = torch.zeros(130, 300).to(torch.float8_e4m3fn)


def test_uncast_takes_what_fits(launches):
    for scale, block in ((torch.ones(130, 3), (1, 128)), (torch.ones(2, 300), (128, 1)), (torch.ones(2, 3), (128, 128)),
                         (torch.ones(1, 1).expand(2, 3), (128, 128)), (torch.ones(3, 130).t(), (1, 128))):
        assert _ops._uncast_blockwise_cuda(Q, scale, *block, BF).shape == (130, 300)
        assert _ops._uncast_blockwise_cuda(Q.t(), scale.t(), *block[::-1], BF).shape == (300, 130)
    assert len(launches) == 10


@pytest.mark.parametrize("scale,block,match", [
    (torch.ones(130, 2), (1, 128), "scale_inv must be"), (torch.ones(129, 3), (1, 128), "scale_inv must be"),
    (torch.ones(2, 3), (1, 128), "scale_inv must be"), (torch.ones(130, 3), (128, 128), "scale_inv must be"),
    (torch.ones(6), (128, 128), "scale_inv must be"), (torch.ones(2, 3).half(), (128, 128), "scale_inv must be"),
    (torch.ones(3, 5), (64, 64), "blocks of 1 or 128"),
])
def test_uncast_refuses_what_does_not(launches, scale, block, match):
    with pytest.raises(RuntimeError, match=match):
        _ops._uncast_blockwise_cuda(Q, scale, *block, BF)
    with pytest.raises(RuntimeError, match=match):
        _ops._uncast_blockwise_cuda(Q.t(), scale.t(), *block[::-1], BF)
    with pytest.raises(RuntimeError, match="takes a matrix"):
        _ops._uncast_blockwise_cuda(Q[0], scale, *block, BF)
    assert not launches
