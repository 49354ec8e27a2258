"""Argument checks of the block-scaled casts and products, the layer norm and the gradient norm: nothing here reaches a
kernel, so it runs without a GPU."""
import ctypes

import pytest
import torch

import float8_experimental_b200 as f8
from float8_experimental_b200 import _native as N
from float8_experimental_b200._ops import _check_dense, _exponent_bytes
from float8_experimental_b200.float8_blockwise import (
    blockwise_mm, cast_to_float8_blockwise, cast_to_float8_blockwise_both, Float8BlockTensor,
)
from float8_experimental_b200.float8_linear import Float8Linear

E4 = torch.float8_e4m3fn
vp = ctypes.c_void_p
P, Q = vp(256), vp(4096)


def block_tensor(rows, cols, block):
    nb = tuple(-(-s // b) for s, b in zip((rows, cols), block))
    return Float8BlockTensor(torch.zeros(rows, cols).to(E4), torch.ones(nb), block)


def test_block_tensor_checks_and_transposes():
    t = block_tensor(130, 300, (1, 128))
    assert t.scale_inv.shape == (130, 3) and t.t().block == (128, 1) and t.t().scale_inv.shape == (3, 130)
    assert t.t().data.data_ptr() == t.data.data_ptr()
    with pytest.raises(ValueError, match="block must be"):
        block_tensor(4, 4, (1, 64))
    with pytest.raises(ValueError, match="float8 matrix"):
        Float8BlockTensor(torch.zeros(4, 4), torch.ones(4, 1), (1, 128))
    with pytest.raises(ValueError, match="scale_inv must be"):
        Float8BlockTensor(torch.zeros(4, 4).to(E4), torch.ones(1, 4), (1, 128))
    with pytest.raises(ValueError, match="scale_inv must be"):
        Float8BlockTensor(torch.zeros(4, 4).to(E4), torch.ones(4, 1).half(), (1, 128))


def test_product_and_cast_refusals():
    a, w = block_tensor(4, 256, (1, 128)), block_tensor(8, 256, (128, 128))
    with pytest.raises(TypeError):
        blockwise_mm(a, w.data)
    with pytest.raises(ValueError, match="inner dimensions"):
        blockwise_mm(a, w)
    with pytest.raises(ValueError, match="128 long"):
        blockwise_mm(block_tensor(4, 256, (128, 1)), w.t())
    with pytest.raises(N.F8B200Error):
        blockwise_mm(a, w.t(), out_dtype=torch.float64)
    with pytest.raises(ValueError, match="takes a matrix"):
        cast_to_float8_blockwise(torch.zeros(4))
    with pytest.raises(ValueError, match="block must be"):
        cast_to_float8_blockwise(torch.zeros(4, 4), (128, 64))
    with pytest.raises(ValueError, match="Unsupported float8_dtype"):
        cast_to_float8_blockwise_both(torch.zeros(4, 4), torch.int8)
    with pytest.raises(NotImplementedError):  # no CPU implementation
        cast_to_float8_blockwise(torch.zeros(4, 4))


def test_linear_config_rules():
    blk, dyn = (f8.CastConfig(scaling_type=t) for t in (f8.ScalingType.BLOCKWISE, f8.ScalingType.DYNAMIC))
    lin = torch.nn.Linear(16, 16)
    with pytest.raises(ValueError, match="together"):
        Float8Linear.from_float(lin, f8.Float8LinearConfig(cast_config_input=blk, cast_config_weight=dyn))
    every = dict(cast_config_input=blk, cast_config_weight=blk, cast_config_grad_output=blk)
    with pytest.raises(ValueError, match="per-tensor scale"):
        Float8Linear.from_float(lin, f8.Float8LinearConfig(**every, enable_fsdp_float8_all_gather=True))
    config = f8.Float8LinearConfig(**every)
    layer = Float8Linear.from_float(lin, config)
    assert layer.scaling_repr() == "i:blk,w:blk,go:blk" and not f8.linear_requires_sync(config)
    assert layer.weight is lin.weight and not dict(layer.named_buffers())


def test_layer_norm_module_rules():
    m = f8.LayerNorm(8, bias=False)
    assert m.bias is None and set(m.state_dict()) == {"weight"}
    with pytest.raises(ValueError, match="last dimension only"):
        f8.LayerNorm((4, 8))
    with pytest.raises(RuntimeError, match="must be 8"):
        m(torch.zeros(2, 7))
    with pytest.raises(NotImplementedError):
        m(torch.zeros(2, 8))


def test_grad_clip_rules():
    with pytest.raises(ValueError, match="norm_type"):
        f8.get_total_norm([torch.zeros(3)], 0.5)
    assert float(f8.get_total_norm([])) == 0.0
    assert float(f8.clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0.0
    x = torch.zeros(4, 6, 8)
    _check_dense("t", [x, x.permute(2, 0, 1), x.transpose(0, 1), torch.zeros(3, 1).t(), torch.zeros(0, 3)])
    for bad in (x[:, ::2], x[..., :4], x[:1, :1, :1].expand(2, 1, 1)):
        with pytest.raises(RuntimeError, match="not dense"):
            _check_dense("t", [bad])


def test_c_argument_checks_come_before_any_cuda_call():
    lib = N.load()
    cast = lambda **k: lib.f8b200_cast_blockwise(*{**dict(  # noqa: E731
        x=P, dt=0, rows=4, cols=8, ld=8, kind=0, sq=0, o=P, ldo=8, s=P, lds=4, e=None, oc=None, ldc=0, sc=None, ldsc=0, ec=None,
        st=None), **k}.values())
    for bad in (dict(dt=3), dict(kind=2), dict(x=None), dict(ld=7), dict(o=None), dict(s=None), dict(ldo=7), dict(lds=3),
                dict(rows=-1), dict(oc=P, ldc=8), dict(oc=P, ldc=7, sc=P, ldsc=8), dict(oc=P, ldc=8, sc=P, ldsc=7),
                dict(sq=1, oc=P, ldc=8, sc=P, ldsc=8), dict(sq=1, lds=0), dict(sq=1, e=P), dict(ec=P)):
        assert cast(**bad) == -1, bad
    assert cast(s=vp(258)) == -2 and cast(x=vp(257)) == -2
    assert cast(rows=0) == 0 and cast(cols=0) == 0
    assert cast(rows=1 << 40, cols=1 << 20, ld=1 << 20, ldo=1 << 20, lds=1 << 40) == -6
    assert lib.f8b200_block_exponent_bytes(1, 1) == 1024 and lib.f8b200_block_exponent_bytes(257, 513) == 4096
    assert _exponent_bytes(257, 513) == 4096 and lib.f8b200_block_exponent_bytes(0, 5) == _exponent_bytes(0, 5) == 0
    unc = lambda **k: lib.f8b200_uncast_blockwise(*{**dict(  # noqa: E731
        q=P, kind=0, rows=4, cols=8, ld=8, s=P, sr=1, sc=1, br=1, bc=128, dt=0, y=P, ldy=8, st=None), **k}.values())
    for bad in (dict(q=None), dict(s=None), dict(y=None), dict(br=2), dict(bc=64), dict(ld=7), dict(ldy=7), dict(sr=-1),
                dict(dt=5), dict(kind=9)):
        assert unc(**bad) == -1, bad
    assert unc(y=vp(257)) == -2 and unc(rows=0) == 0
    mm = lambda **k: lib.f8b200_gemm_blockwise(*{**dict(  # noqa: E731
        a=P, ak=0, al=0, lda=16, sa=P, sar=1, sak=1, ab=1, ea=None, b=P, bk=0, bl=0, ldb=16, sb=P, sbr=1, sbk=1, bb=128, eb=None, bias=None,
        dt=0, out=P, ldo=4, m=4, n=4, k=16, ws=None, wsb=0, st=None), **k}.values())
    assert mm(m=0) == 0 and mm(n=0) == 0 and mm(k=0) == -6
    assert mm(lda=24) == -2 and mm(a=vp(264)) == -2
    assert mm(a=None) == -1 and mm(sa=None) == -1 and mm(ldo=3) == -1 and mm(dt=3) == -1 and mm(k=-1) == -1
    assert mm(ab=2) == -1 and mm(bb=64) == -1 and mm(sar=-1) == -1 and mm(sbk=-1) == -1
    assert mm(ws=Q, wsb=255) == -1 and mm(ws=vp(4104), wsb=256) == -2
    ln = lambda **k: lib.f8b200_layer_norm(*{**dict(  # noqa: E731
        x=P, dt=0, rows=4, cols=8, ld=8, w=P, b=P, at=0, eps=1e-5, y=P, ldy=8, mean=None, rstd=None, st=None), **k}.values())
    for bad in (dict(x=None), dict(y=None), dict(cols=0), dict(rows=-1), dict(ld=7), dict(ldy=7), dict(at=1), dict(dt=4),
                dict(mean=P)):
        assert ln(**bad) == -1, bad
    assert ln(rows=0) == 0 and ln(w=vp(257)) == -2
    bwd = lambda **k: lib.f8b200_layer_norm_bwd(*{**dict(  # noqa: E731
        x=P, g=P, dt=0, rows=4, cols=8, ldx=8, ldg=8, w=P, at=0, mean=P, rstd=P, dx=P, lddx=8, dw=P, db=P, ws=Q,
        wsb=1 << 30, st=None), **k}.values())
    need = lib.f8b200_layer_norm_bwd_workspace_bytes(8)
    for bad in (dict(x=None), dict(g=None), dict(mean=None), dict(rstd=None), dict(ws=None), dict(wsb=need - 1), dict(lddx=7),
                dict(ldg=7), dict(rows=0)):
        assert bwd(**bad) == -1, bad
    assert bwd(ws=vp(4100)) == -2
    ptrs, numels, codes = (vp * 2)(256, 512), (ctypes.c_int64 * 2)(5, 0), (ctypes.c_int * 2)(0, 2)
    assert lib.f8b200_multi_norm_workspace_bytes(numels, 2) == 8
    norm = lambda **k: lib.f8b200_multi_norm(*{**dict(  # noqa: E731
        p=ptrs, n=numels, c=codes, cnt=2, kind=2, root=1, out=P, ws=Q, wsb=8, st=None), **k}.values())
    for bad in (dict(kind=3), dict(out=None), dict(ws=None), dict(wsb=7), dict(cnt=-1), dict(p=None),
                dict(c=(ctypes.c_int * 2)(7, 0)), dict(n=(ctypes.c_int64 * 2)(-1, 0))):
        assert norm(**bad) == -1, bad
    assert norm(ws=vp(4100)) == -2 and norm(p=(vp * 2)(257, 0)) == -2
    assert lib.f8b200_multi_clip(ptrs, numels, codes, 2, None, 1.0, None) == -1
