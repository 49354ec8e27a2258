"""`torch.library` registration of the sm_100a kernels as opaque custom ops.

The reference registers its one private op the same way
(float8_experimental/float8_aten_api.py:37-49: `Library(...)`, `define`, `impl`).
Only a CUDA implementation (and a Meta/fake one for tracing) is registered: calling an
op with CPU tensors fails in the dispatcher, there is no fallback.

Ops (namespace `f8b200`):
  amax(x) -> fp32 0-dim                                   f8b200_amax
  multi_amax(xs) -> fp32 [n]                              f8b200_multi_amax
  amax_to_scale(amax, kind, amax_dtype, orig_dtype)       f8b200_amax_to_scale
  cast_from_amax(x, amax, kind, with_t) -> (data, data_t, scale)   f8b200_cast, scale_src=1
  cast_with_scale(x, scale, kind, product_fp32, with_t, amax_out!) -> (data, data_t)
  cast_dynamic(x, kind) -> (data, scale)                  f8b200_cast_dynamic (amax + cast, one call)
  multi_cast_with_scales(xs, scales, kind, product_fp32) -> fp8 tensors   f8b200_multi_cast
  transpose_fp8(x) -> x^T contiguous                      f8b200_transpose_u8
  delayed_sync(amax, hist, n_e4m3, orig_dtype, scale_out!, hist_out!)
  scaled_mm(a, b_t, scale_a, scale_b, bias, out_dtype, use_fast_accum) -> out
  rmsnorm_amax(x, weight, eps) -> (rstd fp32 [rows], amax fp32 0-dim)      f8b200_rmsnorm_amax
  rmsnorm_cast(x, weight, rstd, amax, kind) -> (data, scale)               f8b200_rmsnorm_cast
  swiglu_amax(a, b, write_y, approx) -> (amax fp32 0-dim, y or empty)      f8b200_swiglu_amax[_approx]
  swiglu_cast(a, b, amax, kind) -> (data, scale)                           f8b200_swiglu_cast
  cast_blockwise(x, kind, by_row, by_col) -> (data, scale_inv, exps, data_c, scale_inv_c, exps_c)
                                                                           f8b200_cast_blockwise
  cast_blockwise_square(x, kind) -> (data, scale_inv, exps, exps_t)        f8b200_cast_blockwise, 128 x 128 blocks
  uncast_blockwise(q, scale_inv, block_rows, block_cols, dtype) -> y       f8b200_uncast_blockwise
  blockwise_mm(a, b_t, scale_a, scale_b, a_block_rows, b_block_rows, exp_a, exp_b, bias, out_dtype) -> out
                                                                           f8b200_gemm_blockwise
  layer_norm(x, weight, bias, eps, save_stats) -> (y, mean, rstd)          f8b200_layer_norm
  layer_norm_bwd(x, grad_y, weight, mean, rstd, affine_dtype, need_dx, need_dw, need_db) -> (dx, dw, db)
  multi_norm(xs, kind, root) -> fp32 0-dim                                 f8b200_multi_norm
  multi_clip_(xs!, total_norm, max_norm)                                   f8b200_multi_clip
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _native as N

_lib = torch.library.Library("f8b200", "DEF")

_lib.define("amax(Tensor x) -> Tensor")
_lib.define("multi_amax(Tensor[] xs) -> Tensor")
_lib.define("amax_to_scale(Tensor amax, int fp8_kind, int amax_dtype, int orig_dtype) -> Tensor")
_lib.define("cast_from_amax(Tensor x, Tensor amax, int fp8_kind, bool with_transpose) -> (Tensor, Tensor, Tensor)")
_lib.define(
    "cast_with_scale(Tensor x, Tensor scale, int fp8_kind, bool product_fp32, bool with_transpose, "
    "Tensor(a!)? amax_out) -> (Tensor, Tensor)"
)
_lib.define("cast_dynamic(Tensor x, int fp8_kind) -> (Tensor, Tensor)")
_lib.define("multi_cast_with_scales(Tensor[] xs, Tensor scales, int fp8_kind, bool product_fp32) -> Tensor[]")
_lib.define("transpose_fp8(Tensor x) -> Tensor")
_lib.define(
    "delayed_sync(Tensor amax, Tensor hist, int n_e4m3, int orig_dtype, Tensor(a!) scale_out, "
    "Tensor(b!)? hist_out) -> ()"
)
_lib.define(
    "scaled_mm(Tensor a, Tensor b_t, Tensor scale_a, Tensor scale_b, Tensor? bias, ScalarType out_dtype, "
    "bool use_fast_accum) -> Tensor"
)
_lib.define("rmsnorm_amax(Tensor x, Tensor weight, float eps) -> (Tensor, Tensor)")
_lib.define("rmsnorm_cast(Tensor x, Tensor weight, Tensor rstd, Tensor amax, int fp8_kind) -> (Tensor, Tensor)")
_lib.define("swiglu_amax(Tensor a, Tensor b, bool write_y, bool approx=False) -> (Tensor, Tensor)")
_lib.define("rmsnorm_bwd(Tensor x, Tensor grad_y, Tensor weight, Tensor rstd) -> (Tensor, Tensor)")
_lib.define("swiglu_bwd(Tensor a, Tensor b, Tensor grad_y, bool approx=False) -> (Tensor, Tensor)")
_lib.define("swiglu_cast(Tensor a, Tensor b, Tensor amax, int fp8_kind) -> (Tensor, Tensor)")
_lib.define("cast_blockwise(Tensor x, int fp8_kind, bool by_row, bool by_col) -> "
            "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)")
_lib.define("cast_blockwise_square(Tensor x, int fp8_kind) -> (Tensor, Tensor, Tensor, Tensor)")
_lib.define("uncast_blockwise(Tensor q, Tensor scale_inv, int block_rows, int block_cols, ScalarType dtype) -> Tensor")
_lib.define(
    "blockwise_mm(Tensor a, Tensor b_t, Tensor scale_a, Tensor scale_b, int a_block_rows, int b_block_rows, "
    "Tensor? exp_a, Tensor? exp_b, Tensor? bias, ScalarType out_dtype) -> Tensor"
)
_lib.define(
    "layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool save_stats) -> (Tensor, Tensor, Tensor)"
)
_lib.define(
    "layer_norm_bwd(Tensor x, Tensor grad_y, Tensor? weight, Tensor mean, Tensor rstd, ScalarType affine_dtype, "
    "bool need_dx, bool need_dw, bool need_db) -> (Tensor, Tensor, Tensor)"
)
_lib.define("multi_norm(Tensor[] xs, int kind, bool root) -> Tensor")
_lib.define("multi_clip_(Tensor(a!)[] xs, Tensor total_norm, float max_norm) -> ()")


def _as_matrix(x: torch.Tensor) -> Tuple[torch.Tensor, int, int, int]:
    """Views `x` as [rows, cols] with unit inner stride; returns (tensor, rows, cols, ld)."""
    cols = x.shape[-1] if x.dim() > 0 else 1
    rows = x.numel() // cols if cols > 0 else 0
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= max(cols, 1):
        return x, rows, cols, x.stride(0)
    if not x.is_contiguous():
        x = x.contiguous()
    return x, rows, cols, cols


def _empty_like_shape(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return torch.empty(x.shape, dtype=dtype, device=x.device)


# ---------------------------------------------------------------------------
# CUDA implementations
# ---------------------------------------------------------------------------
def _amax_cuda(x: torch.Tensor) -> torch.Tensor:
    if x.numel() == 0:
        raise RuntimeError("amax of an empty tensor is undefined")
    if not x.is_contiguous():
        x = x.contiguous()
    out = torch.empty((), dtype=torch.float32, device=x.device)
    N.amax(x, out)
    return out


def _multi_amax_cuda(xs: List[torch.Tensor]) -> torch.Tensor:
    xs = [t if t.is_contiguous() else t.contiguous() for t in xs]
    dev = xs[0].device if xs else torch.device("cuda")
    out = torch.empty((len(xs),), dtype=torch.float32, device=dev)
    N.multi_amax(xs, out)
    return out


def _amax_to_scale_cuda(amax: torch.Tensor, fp8_kind: int, amax_dtype: int, orig_dtype: int) -> torch.Tensor:
    a = amax if (amax.dtype == torch.float32 and amax.is_contiguous()) else amax.float().contiguous()
    out = torch.empty(amax.shape, dtype=torch.float32, device=amax.device)
    N.amax_to_scale(a, fp8_kind, amax_dtype, orig_dtype, out)
    return out


def _alloc_cast_outputs(x: torch.Tensor, rows: int, cols: int, fp8_kind: int, with_transpose: bool):
    f8 = N.FP8_DTYPE[fp8_kind]
    data = _empty_like_shape(x, f8)
    if with_transpose:
        data_t = torch.empty((cols, rows), dtype=f8, device=x.device)
    else:
        data_t = torch.empty((0,), dtype=f8, device=x.device)
    return data, data_t


def _cast_from_amax_cuda(x, amax, fp8_kind: int, with_transpose: bool):
    xm, rows, cols, ld = _as_matrix(x)
    data, data_t = _alloc_cast_outputs(x, rows, cols, fp8_kind, with_transpose)
    scale = torch.empty((), dtype=torch.float32, device=x.device)
    N.cast(xm, rows, cols, ld, 1, amax, scale, False, fp8_kind, data, cols,
           data_t if with_transpose else None, rows, None, True)
    return data, data_t, scale


def _cast_with_scale_cuda(x, scale, fp8_kind: int, product_fp32: bool, with_transpose: bool, amax_out):
    xm, rows, cols, ld = _as_matrix(x)
    data, data_t = _alloc_cast_outputs(x, rows, cols, fp8_kind, with_transpose)
    s = scale if scale.dtype == torch.float32 else scale.float()
    N.cast(xm, rows, cols, ld, 0, s, None, product_fp32, fp8_kind, data, cols,
           data_t if with_transpose else None, rows, amax_out, False)
    return data, data_t


def _cast_dynamic_cuda(x, fp8_kind: int):
    """amax + cast with the scale derived from the amax, one host call: (fp8 data, scale)."""
    if not x.is_contiguous():
        x = x.contiguous()
    cols = x.shape[-1] if x.dim() > 0 else 1
    rows = x.numel() // cols if cols > 0 else 0
    if rows == 0 or cols == 0:
        raise RuntimeError("amax of an empty tensor is undefined")
    data = torch.empty(x.shape, dtype=N.FP8_DTYPE[fp8_kind], device=x.device)
    amax_scale = torch.empty(2, dtype=torch.float32, device=x.device)
    N.cast_dynamic(x, rows, cols, fp8_kind, amax_scale[0], amax_scale[1], data)
    return data, amax_scale[1]


def _multi_cast_with_scales_cuda(xs: List[torch.Tensor], scales: torch.Tensor, fp8_kind: int, product_fp32: bool):
    xs = [t if t.is_contiguous() else t.contiguous() for t in xs]
    s = scales if (scales.dtype == torch.float32 and scales.is_contiguous()) else scales.float().contiguous()
    outs = [torch.empty(t.shape, dtype=N.FP8_DTYPE[fp8_kind], device=t.device) for t in xs]
    N.multi_cast(xs, s, product_fp32, fp8_kind, outs)
    return outs


def _transpose_fp8_cuda(x: torch.Tensor) -> torch.Tensor:
    assert x.dim() == 2
    if x.stride(1) != 1:
        x = x.contiguous()
    rows, cols = x.shape
    out = torch.empty((cols, rows), dtype=x.dtype, device=x.device)
    N.transpose_u8(x, rows, cols, x.stride(0), out, rows)
    return out


def _delayed_sync_cuda(amax, hist, n_e4m3: int, orig_dtype: int, scale_out, hist_out) -> None:
    N.delayed_sync(amax, hist, n_e4m3, orig_dtype, scale_out, hist_out)


def _pitch16(n: int) -> int:
    return -(-n // 16) * 16


def _gemm_operand(x: torch.Tensor):
    """How the GEMM can read the logical [rows, K] operand `x` where it lies: (tensor, pitch,
    mn_major).  K contiguous = K-major; rows contiguous (a transposed view of a [K, rows]
    buffer) = MN-major, which the tensor cores read through an MN-major descriptor.  Anything
    else, or a pitch / base address that TMA cannot take, is copied into a K-major buffer
    whose row pitch is rounded up to 16 bytes.  K itself may be any number: TMA zero-fills
    beyond it, so no operand is ever zero-padded along K (the reference pads both operands
    with a copy when K is not a multiple of 16, float8_experimental/float8_ops.py:143-148)."""
    rows, k = x.shape
    if x.stride(1) == 1 and (rows == 1 or (x.stride(0) >= k and x.stride(0) % 16 == 0)) and x.data_ptr() % 16 == 0:
        return x, (x.stride(0) if rows > 1 else _pitch16(k)), False
    if x.stride(0) == 1 and k > 1 and x.stride(1) >= rows and x.stride(1) % 16 == 0 and x.data_ptr() % 16 == 0:
        return x, x.stride(1), True
    buf = torch.empty((rows, _pitch16(k)), dtype=torch.uint8, device=x.device)
    view = buf[:, :k]
    view.copy_(x.view(torch.uint8))
    return view.view(x.dtype), buf.stride(0), False


def _scaled_mm_cuda(a, b_t, scale_a, scale_b, bias, out_dtype, use_fast_accum: bool):
    m, k = a.shape
    n, k2 = b_t.shape
    if k != k2:
        raise RuntimeError(f"scaled_mm: inner dimensions differ ({k} vs {k2})")
    a, lda, a_mn = _gemm_operand(a)
    b_t, ldb, b_mn = _gemm_operand(b_t)
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    if bias is not None and bias.dtype != out_dtype:
        bias = bias.to(out_dtype)
    sa = scale_a if scale_a.dtype == torch.float32 else scale_a.float()
    sb = scale_b if scale_b.dtype == torch.float32 else scale_b.float()
    N.gemm_fp8(a, lda, b_t, ldb, sa, sb, bias, out, n, m, n, k, use_fast_accum, a_mn_major=a_mn, b_mn_major=b_mn)
    return out


def _rmsnorm_amax_cuda(x, weight, eps: float):
    xm, rows, cols, ld = _as_matrix(x)
    weight = weight.contiguous()
    if weight.dtype != x.dtype or weight.numel() != cols:
        raise RuntimeError("rmsnorm_amax: the weight must have x's dtype and one element per column")
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    amax = torch.empty((), dtype=torch.float32, device=x.device)
    N.rmsnorm_amax(xm, rows, cols, ld, weight, eps, rstd, amax)
    return rstd, amax


def _rmsnorm_cast_cuda(x, weight, rstd, amax, fp8_kind: int):
    xm, rows, cols, ld = _as_matrix(x)
    weight = weight.contiguous()
    data = _empty_like_shape(x, N.FP8_DTYPE[fp8_kind])
    scale = torch.empty((), dtype=torch.float32, device=x.device)
    N.rmsnorm_cast(xm, rows, cols, ld, weight, rstd, amax, scale, data, cols)
    return data, scale


def _glu_operands(a, b):
    if a.shape != b.shape or a.dtype != b.dtype:
        raise RuntimeError("swiglu: a and b must have one shape and dtype")
    am, rows, cols, lda = _as_matrix(a)
    bm, _, _, ldb = _as_matrix(b)
    return am, bm, rows, cols, lda, ldb


def _swiglu_amax_cuda(a, b, write_y: bool, approx: bool = False):
    am, bm, rows, cols, lda, ldb = _glu_operands(a, b)
    amax = torch.empty((), dtype=torch.float32, device=a.device)
    y = _empty_like_shape(a, a.dtype) if write_y else a.new_empty((0,))
    N.swiglu_amax(am, bm, rows, cols, lda, ldb, y if write_y else None, cols, amax, approx)
    return amax, y


def _swiglu_cast_cuda(a, b, amax, fp8_kind: int):
    am, bm, rows, cols, lda, ldb = _glu_operands(a, b)
    data = _empty_like_shape(a, N.FP8_DTYPE[fp8_kind])
    scale = torch.empty((), dtype=torch.float32, device=a.device)
    N.swiglu_cast(am, bm, rows, cols, lda, ldb, amax, scale, data, cols)
    return data, scale


def _rmsnorm_bwd_cuda(x, grad_y, weight, rstd):
    xm, rows, cols, ld = _as_matrix(x.contiguous())
    gm, _, _, ldg = _as_matrix(grad_y.contiguous())
    dx = torch.empty_like(xm)
    dw = torch.empty_like(weight)
    N.rmsnorm_bwd(xm, gm, rows, cols, ld, ldg, weight.contiguous(), rstd, dx, dw)
    return dx.view(x.shape), dw


def _swiglu_bwd_cuda(a, b, grad_y, approx: bool = False):
    am, bm, rows, cols, lda, ldb = _glu_operands(a, b)
    gm, _, _, ldg = _as_matrix(grad_y.reshape(a.shape).contiguous())
    da = torch.empty(a.shape, dtype=a.dtype, device=a.device)
    db = torch.empty(a.shape, dtype=a.dtype, device=a.device)
    N.swiglu_bwd(am, bm, gm, rows, cols, lda, ldb, ldg, da, db, approx)
    return da, db


def _one_device(what: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise RuntimeError(f"{what}: tensors on different devices ({device} and {t.device})")


def _blocks(size: int) -> int:
    return -(-size // 128)


def _empty_fp8_matrix(rows: int, cols: int, fp8_kind: int, device) -> torch.Tensor:
    """[rows, cols] fp8 whose rows start on 16-byte boundaries, so that the GEMM reads it where it lies."""
    out = torch.empty((rows, _pitch16(cols)), dtype=N.FP8_DTYPE[fp8_kind], device=device)
    return out if cols % 16 == 0 else out[:, :cols]


def _exponent_bytes(rows: int, k: int) -> int:
    """f8b200_block_exponent_bytes: four k-blocks to a word, the rows rounded up to a tile of 256."""
    return -(-rows // 256) * 1024 * -(-k // 512)


def _cast_blockwise_some(x, fp8_kind: int, by_row: bool, by_col: bool):
    """The forms asked for as (data, scale_inv, exps), None for the others."""
    if x.dim() != 2 or not (by_row or by_col):
        raise RuntimeError("cast_blockwise: takes a matrix and at least one of by_row, by_col")
    xm, _, _, ld = _as_matrix(x)
    rows, cols = x.shape
    device = x.device

    def form(n, k):  # one factor per (block, row) resp. (block, column): the GEMM's lanes read neighbouring rows
        data = _empty_fp8_matrix(rows, cols, fp8_kind, device)
        scale = torch.empty((_blocks(k), n), dtype=torch.float32, device=device)
        return data, scale, torch.empty(_exponent_bytes(n, k), dtype=torch.uint8, device=device)

    r = form(rows, cols) if by_row else None
    c = form(cols, rows) if by_col else None
    if rows and cols:
        N.cast_blockwise(xm, rows, cols, ld, fp8_kind, False,
                         *((r[0], r[0].stride(0), r[1], rows, r[2]) if by_row else (None, 0, None, 0, None)),
                         *((c[0], c[0].stride(0), c[1], cols, c[2]) if by_col else (None, 0, None, 0, None)))
    return (r[0], r[1].t(), r[2]) if by_row else (None, None, None), c if by_col else (None, None, None)


def _cast_blockwise_cuda(x, fp8_kind: int, by_row: bool, by_col: bool):
    r, c = _cast_blockwise_some(x, fp8_kind, by_row, by_col)

    def none():
        return (torch.empty((0, 0), dtype=N.FP8_DTYPE[fp8_kind], device=x.device),
                torch.empty((0, 0), dtype=torch.float32, device=x.device),
                torch.empty((0,), dtype=torch.uint8, device=x.device))

    return (*(r if by_row else none()), *(c if by_col else none()))


def _cast_blockwise_square_cuda(x, fp8_kind: int):
    if x.dim() != 2:
        raise RuntimeError("cast_blockwise_square: takes a matrix")
    xm, _, _, ld = _as_matrix(x)
    rows, cols = x.shape
    data = _empty_fp8_matrix(rows, cols, fp8_kind, x.device)
    scale = torch.empty((_blocks(rows), _blocks(cols)), dtype=torch.float32, device=x.device)
    exps, exps_t = (torch.empty(_exponent_bytes(r, c), dtype=torch.uint8, device=x.device)
                    for r, c in ((rows, cols), (cols, rows)))
    if x.numel():
        N.cast_blockwise(xm, rows, cols, ld, fp8_kind, True, data, data.stride(0), scale, scale.shape[1], exps,
                         None, 0, None, 0, exps_t)
    return data, scale, exps, exps_t


_BLOCK_SIZES = (1, 128)


def _uncast_blockwise_cuda(q, scale_inv, block_rows: int, block_cols: int, dtype):
    if q.dim() != 2 or block_rows not in _BLOCK_SIZES or block_cols not in _BLOCK_SIZES:
        raise RuntimeError("uncast_blockwise: takes a matrix in blocks of 1 or 128 each way")
    rows, cols = q.shape
    want = (-(-rows // block_rows), -(-cols // block_cols))
    if scale_inv.dtype is not torch.float32 or scale_inv.shape != want:
        raise RuntimeError(f"uncast_blockwise: scale_inv must be float32 {want}, got {scale_inv.dtype} {tuple(scale_inv.shape)}")
    _one_device("uncast_blockwise", q, scale_inv)
    if rows != 1 and cols != 1 and q.stride(0) == 1:  # a transposed matrix: read it as it lies
        return _uncast_blockwise_cuda(q.t(), scale_inv.t(), block_cols, block_rows, dtype).t()
    if q.stride(1) != 1 or q.stride(0) < cols:
        q = q.contiguous()
    y = torch.empty((rows, cols), dtype=dtype, device=q.device)
    if q.numel():
        N.uncast_blockwise(q, rows, cols, max(q.stride(0), cols), scale_inv, block_rows, block_cols, y, cols)
    return y


def _check_factors(name: str, s, rows: int, k: int, block: int) -> None:
    if s.dtype != torch.float32 or s.shape != (-(-rows // 128) if block == 128 else rows, -(-k // 128)):
        want = (_blocks(rows) if block == 128 else rows, _blocks(k))
        raise RuntimeError(f"blockwise_mm: {name} must be float32 {want}, got {s.dtype} {tuple(s.shape)}")


def _dense_bias(bias: Optional[torch.Tensor], n: int, dtype: torch.dtype) -> Optional[torch.Tensor]:
    """The bias as the products read it: n neighbouring elements of the result's type."""
    if bias is None:
        return None
    if bias.shape != (n,):
        raise RuntimeError(f"blockwise_mm: the bias must have {n} elements, got {tuple(bias.shape)}")
    return bias.to(dtype).contiguous()


def _blockwise_mm_cuda(a, b_t, scale_a, scale_b, a_block_rows: int, b_block_rows: int, exp_a, exp_b, bias, out_dtype):
    _one_device("blockwise_mm", a, b_t, scale_a, scale_b, exp_a, exp_b, bias)
    m, k = a.shape
    n, k2 = b_t.shape
    if k != k2:
        raise RuntimeError(f"blockwise_mm: inner dimensions differ ({k} vs {k2})")
    _check_factors("scale_a", scale_a, m, k, a_block_rows)
    _check_factors("scale_b", scale_b, n, k, b_block_rows)
    for name, e, rows in (("exp_a", exp_a, m), ("exp_b", exp_b, n)):
        if e is not None and (e.dtype != torch.uint8 or not e.is_contiguous() or e.numel() != _exponent_bytes(rows, k)):
            raise RuntimeError(f"blockwise_mm: {name} must be the {_exponent_bytes(rows, k)} exponent bytes of its cast")
    bias = _dense_bias(bias, n, out_dtype)
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    if m == 0 or n == 0:
        return out
    if k == 0:
        return out.zero_() if bias is None else out.copy_(bias)
    a, lda, a_mn = _gemm_operand(a)
    b_t, ldb, b_mn = _gemm_operand(b_t)
    N.gemm_blockwise(a, lda, a_mn, scale_a, a_block_rows, exp_a, b_t, ldb, b_mn, scale_b, b_block_rows, exp_b, bias, out, n,
                     m, n, k)
    return out


def linear_blockwise(x, weight, weight_scale, bias):
    """x [m, k] cast by rows times the transpose of `weight` [n, k] (fp8, `weight_scale` per 128 x 128), plus bias: eager
    CUDA tensors, without autograd."""
    m, k = x.shape
    n, k2 = weight.shape
    if k != k2:
        raise RuntimeError(f"blockwise_mm: inner dimensions differ ({k} vs {k2})")
    if weight_scale.dtype != torch.float32 or tuple(weight_scale.shape) != (_blocks(n), _blocks(k)):
        raise RuntimeError(f"blockwise_mm: scale_b must be float32 {(_blocks(n), _blocks(k))}, got {weight_scale.dtype} "
                           f"{tuple(weight_scale.shape)}")
    _one_device("blockwise_mm", x, weight, weight_scale, bias)
    bias = _dense_bias(bias, n, x.dtype)
    out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    if m == 0 or n == 0:
        return out
    if k == 0:
        return out.zero_() if bias is None else out.copy_(bias)
    xm, _, _, ld = _as_matrix(x)
    weight, ldw, w_mn = _gemm_operand(weight)
    N.linear_blockwise(xm, m, k, ld, weight, ldw, w_mn, weight_scale, bias, out, n)
    return out


def _affine_dtype(x, weight, bias) -> torch.dtype:
    """The type of the norm's weight and bias: x's or fp32, the same for both."""
    first = weight if weight is not None else bias
    if first is None:
        return x.dtype
    affine, want = first.dtype, x.shape[-1:]
    if (affine != x.dtype and affine != torch.float32) or (bias is not None and bias.dtype != affine):
        raise RuntimeError(f"layer_norm: weight and bias must both have x's dtype {x.dtype} or both float32")
    if first.shape != want or (bias is not None and bias.shape != want):
        raise RuntimeError(f"layer_norm: weight and bias must have one element per column ({want[0]})")
    return affine


def layer_norm_into(x, weight, bias, eps: float, mean, rstd):
    """y, and the rows' mean and 1/std when they are asked for: eager CUDA tensors, without autograd."""
    _one_device("layer_norm", x, weight, bias)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError("layer_norm: the last dimension must have at least one element")
    affine = _affine_dtype(x, weight, bias)
    xm, rows, cols, ld = _as_matrix(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if rows:
        N.layer_norm(xm, rows, cols, ld, None if weight is None else weight.contiguous(),
                     None if bias is None else bias.contiguous(), affine, eps, y, mean, rstd)
    return y


def _layer_norm_cuda(x, weight, bias, eps: float, save_stats: bool):
    rows = x.numel() // x.shape[-1] if save_stats and x.dim() and x.shape[-1] else 0
    # two tensors of their own: views of one would share its version counter and outlive it together
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    y = layer_norm_into(x, weight, bias, eps, mean if save_stats else None, rstd if save_stats else None)
    return y, mean, rstd


def _refuse_layer_norm_bwd(x, grad_y, weight, mean, rstd, affine_dtype, rows: int):
    """Says what of the arguments does not fit."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError("layer_norm_bwd: the last dimension must have at least one element")
    if grad_y.shape != x.shape or grad_y.dtype != x.dtype:
        raise RuntimeError(f"layer_norm_bwd: grad_y must be like x, {x.dtype} {tuple(x.shape)}, got {grad_y.dtype} "
                           f"{tuple(grad_y.shape)}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.shape != (rows,) or not t.is_contiguous():
            raise RuntimeError(f"layer_norm_bwd: {name} must be {rows} contiguous float32 values, got {t.dtype} "
                               f"{tuple(t.shape)} with strides {t.stride()}")
    _affine_dtype(x, weight, None)
    raise RuntimeError(f"layer_norm_bwd: affine_dtype {affine_dtype} is not that of the weight and the bias")


def _layer_norm_bwd_cuda(x, grad_y, weight, mean, rstd, affine_dtype, need_dx: bool, need_dw: bool, need_db: bool):
    _one_device("layer_norm_bwd", x, grad_y, weight, mean, rstd)
    xm, rows, cols, ld = _as_matrix(x)
    f32, dtype, stats = torch.float32, x.dtype, (rows,)
    fits = (cols > 0 and x.dim() > 0 and grad_y.shape == x.shape and grad_y.dtype is dtype
            and mean.shape == stats and rstd.shape == stats and mean.dtype is f32 and rstd.dtype is f32 and mean.is_contiguous() and rstd.is_contiguous()
            and (affine_dtype is dtype or affine_dtype is f32)
            and (weight is None or (weight.dtype is affine_dtype and weight.shape == (cols,))))
    if not fits:
        _refuse_layer_norm_bwd(x, grad_y, weight, mean, rstd, affine_dtype, rows)
    gm, _, _, ldg = _as_matrix(grad_y)
    dx = _empty_like_shape(x, x.dtype) if need_dx else x.new_empty((0,))
    # no rows: nothing to sum
    new = torch.empty if rows else torch.zeros
    dw = new((cols if need_dw else 0,), dtype=affine_dtype, device=x.device)
    db = new((cols if need_db else 0,), dtype=affine_dtype, device=x.device)
    if rows and (need_dx or need_dw or need_db):
        N.layer_norm_bwd(xm, gm, rows, cols, ld, ldg, None if weight is None else weight.contiguous(), affine_dtype,
                         mean, rstd, dx if need_dx else None, dw if need_dw else None, db if need_db else None)
    return dx, dw, db


def _check_dense(what: str, xs: List[torch.Tensor]) -> None:
    """The kernels walk a tensor's storage: its elements must fill a range of it, each once, in any order."""
    if all(map(torch.Tensor.is_contiguous, xs)):
        return
    for t in xs:
        if t.is_contiguous():
            continue
        step = 1
        for size, stride in sorted(zip(t.shape, t.stride()), key=lambda d: d[1]):
            if size == 1:
                continue
            if stride != step:
                raise RuntimeError(f"{what}: a tensor of shape {tuple(t.shape)} and strides {t.stride()} is not dense")
            step *= size


class TensorList(N.TensorArrays):
    """Checked arguments of the multi-tensor kernels, made once for the calls that share the tensors."""

    def __init__(self, what: str, xs: List[torch.Tensor]):
        super().__init__(xs)
        _check_dense(what, xs)


def _multi_norm_cuda(xs: List[torch.Tensor], kind: int, root: bool):
    out = torch.empty((), dtype=torch.float32, device=xs[0].device if xs else torch.device("cuda"))
    N.multi_norm(TensorList("multi_norm", xs), kind, root, out)
    return out


def _multi_clip_cuda(xs: List[torch.Tensor], total_norm, max_norm: float) -> None:
    tensors = TensorList("multi_clip_", xs)
    if tensors.device not in (None, total_norm.device):
        raise RuntimeError(f"multi_clip_: tensors on different devices ({tensors.device} and {total_norm.device})")
    if total_norm.numel() != 1 or total_norm.dtype != torch.float32:
        raise RuntimeError("multi_clip_: total_norm must be one float32 value")
    N.multi_clip(tensors, total_norm, max_norm)
    increment_version(xs)  # a kernel's writes leave the versions that autograd compares alone


_lib.impl("cast_blockwise", _cast_blockwise_cuda, "CUDA")
_lib.impl("cast_blockwise_square", _cast_blockwise_square_cuda, "CUDA")
_lib.impl("uncast_blockwise", _uncast_blockwise_cuda, "CUDA")
_lib.impl("blockwise_mm", _blockwise_mm_cuda, "CUDA")
_lib.impl("layer_norm", _layer_norm_cuda, "CUDA")
_lib.impl("layer_norm_bwd", _layer_norm_bwd_cuda, "CUDA")
_lib.impl("multi_norm", _multi_norm_cuda, "CUDA")
_lib.impl("multi_clip_", _multi_clip_cuda, "CUDA")
_lib.impl("rmsnorm_bwd", _rmsnorm_bwd_cuda, "CUDA")
_lib.impl("swiglu_bwd", _swiglu_bwd_cuda, "CUDA")
_lib.impl("swiglu_amax", _swiglu_amax_cuda, "CUDA")
_lib.impl("swiglu_cast", _swiglu_cast_cuda, "CUDA")
_lib.impl("rmsnorm_amax", _rmsnorm_amax_cuda, "CUDA")
_lib.impl("rmsnorm_cast", _rmsnorm_cast_cuda, "CUDA")
_lib.impl("amax", _amax_cuda, "CUDA")
_lib.impl("multi_amax", _multi_amax_cuda, "CUDA")
_lib.impl("amax_to_scale", _amax_to_scale_cuda, "CUDA")
_lib.impl("cast_from_amax", _cast_from_amax_cuda, "CUDA")
_lib.impl("cast_with_scale", _cast_with_scale_cuda, "CUDA")
_lib.impl("transpose_fp8", _transpose_fp8_cuda, "CUDA")
_lib.impl("multi_cast_with_scales", _multi_cast_with_scales_cuda, "CUDA")
_lib.impl("cast_dynamic", _cast_dynamic_cuda, "CUDA")
_lib.impl("delayed_sync", _delayed_sync_cuda, "CUDA")
_lib.impl("scaled_mm", _scaled_mm_cuda, "CUDA")


_PLAIN = (torch.Tensor, torch.nn.Parameter)


_is_compiling = torch.compiler.is_compiling
_dispatch_modes = torch._C._len_torch_dispatch_stack
_pre_dispatch_modes = torch._ops.mode_stack_state_for_pre_dispatch().count
_jit_tracing = torch._C._is_tracing
_functorch_level = torch._C._functorch.peek_interpreter_stack


def nothing_watches() -> bool:
    """Whether no trace (`make_fx`, `torch.jit.trace`), dispatch mode (selective checkpointing, counters, fake tensors) or
    functorch transform would have to see the ops that run here.  All of these show plain tensors."""
    return not _dispatch_modes() and not _jit_tracing() and _functorch_level() is None and not _pre_dispatch_modes()


def eager_cuda(t: torch.Tensor) -> bool:
    """Whether an op on `t` would come straight to its CUDA implementation here: a plain CUDA tensor, `nothing_watches`.
    Callers that run without autograd (inside an autograd function, or with nothing to differentiate) then call
    the implementation themselves: a trip through the dispatcher costs more host time than a small launch."""
    # its checks spelt out: one more Python call costs as much as two of them
    return (not _is_compiling() and type(t) in _PLAIN and t.is_cuda
            and not _dispatch_modes() and not _jit_tracing() and _functorch_level() is None and not _pre_dispatch_modes())


# ---------------------------------------------------------------------------
# fake (meta) implementations: shapes and dtypes only, so torch.compile can trace
# around the opaque ops
# ---------------------------------------------------------------------------
@torch.library.register_fake("f8b200::rmsnorm_bwd")
def _rmsnorm_bwd_fake(x, grad_y, weight, rstd):
    return torch.empty_like(x), torch.empty_like(weight)


@torch.library.register_fake("f8b200::swiglu_bwd")
def _swiglu_bwd_fake(a, b, grad_y, approx=False):
    return torch.empty_like(a), torch.empty_like(a)


@torch.library.register_fake("f8b200::swiglu_amax")
def _swiglu_amax_fake(a, b, write_y, approx=False):
    return a.new_empty((), dtype=torch.float32), a.new_empty(a.shape if write_y else (0,))


@torch.library.register_fake("f8b200::swiglu_cast")
def _swiglu_cast_fake(a, b, amax, fp8_kind):
    return a.new_empty(a.shape, dtype=N.FP8_DTYPE[fp8_kind]), a.new_empty((), dtype=torch.float32)


@torch.library.register_fake("f8b200::rmsnorm_amax")
def _rmsnorm_amax_fake(x, weight, eps):
    cols = x.shape[-1]
    return x.new_empty((x.numel() // max(cols, 1),), dtype=torch.float32), x.new_empty((), dtype=torch.float32)


@torch.library.register_fake("f8b200::rmsnorm_cast")
def _rmsnorm_cast_fake(x, weight, rstd, amax, fp8_kind):
    return x.new_empty(x.shape, dtype=N.FP8_DTYPE[fp8_kind]), x.new_empty((), dtype=torch.float32)


@torch.library.register_fake("f8b200::amax")
def _amax_fake(x):
    return x.new_empty((), dtype=torch.float32)


@torch.library.register_fake("f8b200::multi_amax")
def _multi_amax_fake(xs):
    return xs[0].new_empty((len(xs),), dtype=torch.float32)


@torch.library.register_fake("f8b200::amax_to_scale")
def _amax_to_scale_fake(amax, fp8_kind, amax_dtype, orig_dtype):
    return amax.new_empty(amax.shape, dtype=torch.float32)


def _fake_cast_outputs(x, fp8_kind, with_transpose):
    f8 = N.FP8_DTYPE[fp8_kind]
    cols = x.shape[-1] if x.dim() > 0 else 1
    rows = x.numel() // cols if cols > 0 else 0
    data = x.new_empty(x.shape, dtype=f8)
    data_t = x.new_empty((cols, rows) if with_transpose else (0,), dtype=f8)
    return data, data_t


@torch.library.register_fake("f8b200::cast_from_amax")
def _cast_from_amax_fake(x, amax, fp8_kind, with_transpose):
    data, data_t = _fake_cast_outputs(x, fp8_kind, with_transpose)
    return data, data_t, x.new_empty((), dtype=torch.float32)


@torch.library.register_fake("f8b200::cast_with_scale")
def _cast_with_scale_fake(x, scale, fp8_kind, product_fp32, with_transpose, amax_out):
    return _fake_cast_outputs(x, fp8_kind, with_transpose)


@torch.library.register_fake("f8b200::cast_dynamic")
def _cast_dynamic_fake(x, fp8_kind):
    return x.new_empty(x.shape, dtype=N.FP8_DTYPE[fp8_kind]), x.new_empty((), dtype=torch.float32)


@torch.library.register_fake("f8b200::multi_cast_with_scales")
def _multi_cast_with_scales_fake(xs, scales, fp8_kind, product_fp32):
    return [t.new_empty(t.shape, dtype=N.FP8_DTYPE[fp8_kind]) for t in xs]


@torch.library.register_fake("f8b200::transpose_fp8")
def _transpose_fp8_fake(x):
    return x.new_empty((x.shape[1], x.shape[0]))


@torch.library.register_fake("f8b200::delayed_sync")
def _delayed_sync_fake(amax, hist, n_e4m3, orig_dtype, scale_out, hist_out):
    return None


@torch.library.register_fake("f8b200::scaled_mm")
def _scaled_mm_fake(a, b_t, scale_a, scale_b, bias, out_dtype, use_fast_accum):
    return a.new_empty((a.shape[0], b_t.shape[0]), dtype=out_dtype)


@torch.library.register_fake("f8b200::cast_blockwise")
def _cast_blockwise_fake(x, fp8_kind, by_row, by_col):
    rows, cols = x.shape
    f8 = N.FP8_DTYPE[fp8_kind]

    def data(on):
        return x.new_empty((rows, _pitch16(cols)), dtype=f8)[:, :cols] if on else x.new_empty((0, 0), dtype=f8)

    scale = x.new_empty((_blocks(cols), rows) if by_row else (0, 0), dtype=torch.float32)
    scale_c = x.new_empty((_blocks(rows), cols) if by_col else (0, 0), dtype=torch.float32)
    exps = x.new_empty((_exponent_bytes(rows, cols) if by_row else 0,), dtype=torch.uint8)
    exps_c = x.new_empty((_exponent_bytes(cols, rows) if by_col else 0,), dtype=torch.uint8)
    return data(by_row), scale.t(), exps, data(by_col), scale_c, exps_c


@torch.library.register_fake("f8b200::cast_blockwise_square")
def _cast_blockwise_square_fake(x, fp8_kind):
    rows, cols = x.shape
    data = x.new_empty((rows, _pitch16(cols)), dtype=N.FP8_DTYPE[fp8_kind])[:, :cols]
    exps, exps_t = (x.new_empty((_exponent_bytes(r, c),), dtype=torch.uint8) for r, c in ((rows, cols), (cols, rows)))
    return data, x.new_empty((_blocks(rows), _blocks(cols)), dtype=torch.float32), exps, exps_t


@torch.library.register_fake("f8b200::uncast_blockwise")
def _uncast_blockwise_fake(q, scale_inv, block_rows, block_cols, dtype):
    rows, cols = q.shape
    if rows != 1 and cols != 1 and q.stride(0) == 1:  # a transposed matrix stays one
        return q.new_empty((cols, rows), dtype=dtype).t()
    return q.new_empty((rows, cols), dtype=dtype)


@torch.library.register_fake("f8b200::blockwise_mm")
def _blockwise_mm_fake(a, b_t, scale_a, scale_b, a_block_rows, b_block_rows, exp_a, exp_b, bias, out_dtype):
    return a.new_empty((a.shape[0], b_t.shape[0]), dtype=out_dtype)


@torch.library.register_fake("f8b200::layer_norm")
def _layer_norm_fake(x, weight, bias, eps, save_stats):
    rows = x.numel() // max(x.shape[-1], 1) if save_stats else 0
    return x.new_empty(x.shape), x.new_empty((rows,), dtype=torch.float32), x.new_empty((rows,), dtype=torch.float32)


@torch.library.register_fake("f8b200::layer_norm_bwd")
def _layer_norm_bwd_fake(x, grad_y, weight, mean, rstd, affine_dtype, need_dx, need_dw, need_db):
    cols = x.shape[-1]
    return (x.new_empty(x.shape if need_dx else (0,)), x.new_empty((cols if need_dw else 0,), dtype=affine_dtype),
            x.new_empty((cols if need_db else 0,), dtype=affine_dtype))


@torch.library.register_fake("f8b200::multi_norm")
def _multi_norm_fake(xs, kind, root):
    return xs[0].new_empty((), dtype=torch.float32)


@torch.library.register_fake("f8b200::multi_clip_")
def _multi_clip_fake(xs, total_norm, max_norm):
    return None


ops = torch.ops.f8b200
