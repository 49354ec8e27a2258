"""float8 with one scale per block of 128: casts, matrix products and the linear layer's products.

Per-tensor scaling (the reference's only kind, float8_experimental/config.py:12-21) lets one large value push
the rest of its tensor towards the small end of the format.  Here each block of 128 elements has a factor of
its own.  A block is 1 x 128 (by rows: activations and gradients as a product's left operand), 128 x 1 (by
columns: the same two in the product of the weight's gradient, where they are summed over rows) or 128 x 128
(weights, whose bytes then serve a product and its transpose alike).

The cast picks powers of two (`scale_inv = 2^-e`, e the largest whole number that keeps the block's amax within the
format, amaxes below 1e-12 counting as that), so scaling moves exponents only and rounds nothing.  The product takes
any fp32 factors, such as those that came with a checkpoint's weights.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from ._ops import (
    _as_matrix, _blocks, _blockwise_mm_cuda, _cast_blockwise_some, _cast_blockwise_square_cuda, _dense_bias,
    eager_cuda, linear_blockwise, _one_device, ops, _uncast_blockwise_cuda,
)
from .float8_utils import _kind, e4m3_dtype, e5m2_dtype

__all__ = ["BLOCK", "Float8BlockTensor", "cast_to_float8_blockwise", "cast_to_float8_blockwise_both", "blockwise_mm"]

BLOCK = 128
_BLOCKS = ((1, BLOCK), (BLOCK, 1), (BLOCK, BLOCK))


class Float8BlockTensor:
    """A matrix held as fp8 bytes and one factor per block: `data[i, j] * scale_inv[i // block[0], j // block[1]]`.

    data       [rows, cols] torch.float8_e4m3fn or float8_e5m2, in either memory order
    scale_inv  float32 [ceil(rows / block[0]), ceil(cols / block[1])], any strides
    block      (1, 128), (128, 1) or (128, 128); the last block of a dimension may be shorter
    orig_dtype the dtype `to_original_precision` returns by default

    A cast also keeps its power-of-two factors as the exponent bytes that the tensor cores read (of the matrix, and
    of its transpose, as a product's operand).  Whoever asks for `scale_inv` may write to it, in ways that leave no
    trace (a collective, `.data`, another library's kernel), so asking for it drops the bytes, of transposes too: products
    of more than 128 rows then take the factors themselves, in a slower kernel.  `scale_inv` may be assigned."""

    # _exps: [bytes of the matrix, of its transpose], one list for all the tensors that hold the same factors
    __slots__ = ("data", "_scale", "block", "orig_dtype", "_exps", "_transposed")

    def __init__(self, data: torch.Tensor, scale_inv: torch.Tensor, block: Tuple[int, int],
                 orig_dtype: torch.dtype = torch.bfloat16):
        block = tuple(block)
        if block not in _BLOCKS:
            raise ValueError(f"Float8BlockTensor: block must be one of {_BLOCKS}, got {block}")
        if data.dim() != 2 or data.dtype not in (e4m3_dtype, e5m2_dtype):
            raise ValueError(f"Float8BlockTensor: data must be a float8 matrix, got {data.dtype} {tuple(data.shape)}")
        self.data, self.block, self.orig_dtype = data, block, orig_dtype
        self.scale_inv = scale_inv

    @classmethod
    def _of_cast(cls, data, scale_inv, block, orig_dtype, exps, exps_t) -> "Float8BlockTensor":
        """What a cast made: nothing to check, and the exponent bytes beside it."""
        out = object.__new__(cls)
        out.data, out._scale, out.block, out.orig_dtype = data, scale_inv, block, orig_dtype
        out._exps, out._transposed = [exps, exps_t], False
        return out

    @property
    def scale_inv(self) -> torch.Tensor:
        if self._exps is not None:
            self._exps[:] = None, None
        return self._scale

    @scale_inv.setter
    def scale_inv(self, scale_inv: torch.Tensor) -> None:
        want = tuple(_blocks(size) if b == BLOCK else size for size, b in zip(self.data.shape, self.block))
        if scale_inv.dtype != torch.float32 or tuple(scale_inv.shape) != want:
            raise ValueError(
                f"Float8BlockTensor: scale_inv must be float32 {want} for blocks of {self.block}, got "
                f"{scale_inv.dtype} {tuple(scale_inv.shape)}"
            )
        if scale_inv.device != self.data.device:
            raise ValueError(f"Float8BlockTensor: data on {self.data.device}, scale_inv on {scale_inv.device}")
        self._scale, self._exps, self._transposed = scale_inv, None, False

    def _exponents(self, transposed: bool = False) -> Optional[torch.Tensor]:
        """The exponent bytes, unless the factors may have been written to since the cast."""
        if self._exps is None:
            return None
        return self._exps[transposed != self._transposed]

    @property
    def shape(self) -> torch.Size:
        return self.data.shape

    @property
    def device(self) -> torch.device:
        return self.data.device

    def t(self) -> "Float8BlockTensor":
        """The transposed matrix: the same bytes and factors, nothing copied."""
        out = object.__new__(Float8BlockTensor)
        out.data, out._scale, out.block, out.orig_dtype = self.data.t(), self._scale.t(), self.block[::-1], self.orig_dtype
        out._exps, out._transposed = self._exps, not self._transposed
        return out

    def to_original_precision(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        args = (self.data, self._scale, *self.block, dtype or self.orig_dtype)
        return _uncast_blockwise_cuda(*args) if eager_cuda(self.data) else ops.uncast_blockwise(*args)

    def __repr__(self):
        return f"Float8BlockTensor({self.data.dtype}, shape={tuple(self.shape)}, block={self.block})"


def _cast(x, kind: int, by_row: bool, by_col: bool):
    """((data, scale_inv, exps) by rows, the same by columns); a form not asked for is three None."""
    if eager_cuda(x):
        return _cast_blockwise_some(x, kind, by_row, by_col)
    out = ops.cast_blockwise(x, kind, by_row, by_col)
    none = (None, None, None)
    return out[:3] if by_row else none, out[3:] if by_col else none


def _cast_square(x, kind: int):
    return _cast_blockwise_square_cuda(x, kind) if eager_cuda(x) else ops.cast_blockwise_square(x, kind)


def _mm(a, *args):
    return _blockwise_mm_cuda(a, *args) if eager_cuda(a) else ops.blockwise_mm(a, *args)


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    if x.dim() != 2:
        raise ValueError(f"{what}: takes a matrix, got {x.dim()} dimensions")
    N.hp_code(x.dtype)  # bf16, fp16 or fp32
    return x.detach() if x.requires_grad else x


def cast_to_float8_blockwise(x: torch.Tensor, block: Tuple[int, int] = (1, BLOCK),
                             float8_dtype: torch.dtype = e4m3_dtype) -> Float8BlockTensor:
    """`x` [rows, cols] (bf16 / fp16 / fp32) cast with one power-of-two factor per block.  Not differentiable."""
    block = tuple(block)
    if block not in _BLOCKS:
        raise ValueError(f"cast_to_float8_blockwise: block must be one of {_BLOCKS}, got {block}")
    x, kind = _matrix(x, "cast_to_float8_blockwise"), _kind(float8_dtype)
    if block == (BLOCK, BLOCK):
        data, scale, exps, exps_t = _cast_square(x, kind)
    elif block == (1, BLOCK):
        (data, scale, exps), _ = _cast(x, kind, True, False)
        exps_t = None
    else:
        _, (data, scale, exps_t) = _cast(x, kind, False, True)
        exps = None
    return Float8BlockTensor._of_cast(data, scale, block, x.dtype, exps, exps_t)


def cast_to_float8_blockwise_both(x: torch.Tensor, float8_dtype: torch.dtype = e4m3_dtype
                                  ) -> Tuple[Float8BlockTensor, Float8BlockTensor]:
    """`x` cast by rows (1 x 128 blocks) and by columns (128 x 1), from one read of it."""
    x = _matrix(x, "cast_to_float8_blockwise_both")
    (data, scale, exps), (data_c, scale_c, exps_c) = _cast(x, _kind(float8_dtype), True, True)
    return (Float8BlockTensor._of_cast(data, scale, (1, BLOCK), x.dtype, exps, None),
            Float8BlockTensor._of_cast(data_c, scale_c, (BLOCK, 1), x.dtype, None, exps_c))


def blockwise_mm(a: Float8BlockTensor, b: Float8BlockTensor, out_dtype: torch.dtype = torch.bfloat16,
                 bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a [M, K] @ b [K, N] (+ bias [N]), summed in fp32 and rounded once to `out_dtype` (bf16 / fp16 / fp32).

    The blocks must be 128 long in K on both sides: `a` in 1 x 128 or 128 x 128 blocks, `b` in 128 x 1 (the
    transposed form of 1 x 128) or 128 x 128.  Either operand may lie in either memory order, M, K and N are
    free, and either may be e4m3 or e5m2."""
    if not isinstance(a, Float8BlockTensor) or not isinstance(b, Float8BlockTensor):
        raise TypeError("blockwise_mm: both operands must be Float8BlockTensor")
    if a.block[1] != BLOCK or b.block[0] != BLOCK:
        raise ValueError(f"blockwise_mm: blocks must be {BLOCK} long in the inner dimension, got {a.block} and {b.block}")
    if a.shape[1] != b.shape[0]:
        raise ValueError(f"blockwise_mm: inner dimensions differ ({a.shape[1]} vs {b.shape[0]})")
    N.hp_code(out_dtype)
    return _mm(a.data, b.data.t(), a._scale, b._scale.t(), a.block[0], b.block[1], a._exponents(),
               b._exponents(transposed=True), None if bias is None else bias.detach(), out_dtype)


def linear_by_rows(x: torch.Tensor, weight: torch.Tensor, weight_scale_inv: torch.Tensor,
                   bias: Optional[torch.Tensor]) -> torch.Tensor:
    """x [..., K] cast by rows, times the transpose of an fp8 weight [N, K] with factors per 128 x 128 square, plus bias.
    Not differentiable."""
    N.hp_code(x.dtype)
    with torch.no_grad():
        x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        if eager_cuda(x2):
            y = linear_blockwise(x2, weight, weight_scale_inv, bias)
        else:
            (x8, sx, _), _ = _cast(x2, N.E4M3, True, False)
            y = _mm(x8, weight, sx, weight_scale_inv, 1, BLOCK, None, None, bias, x.dtype)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[-1])


@torch._dynamo.allow_in_graph
class _float8_linear_blockwise(torch.autograd.Function):
    """Forward and backward of a Float8Linear whose three tensors are scaled by blocks, on raw tensors.

    All three are e4m3: with a factor per 128 elements the gradient needs no wider range, and e5m2 would cost it a
    bit of precision.  `need_dw` asks the input's cast for the by-column form that the weight's gradient reads."""

    @staticmethod
    def _forward_eager(ctx, x, x2, weight, bias, need_dw: bool):
        """The same launches with the casts laid out in two buffers: one that the backward pass reads, one that it does
        not need."""
        (m, k), n = x2.shape, weight.shape[0]
        x2, _, _, ldx = _as_matrix(x2)
        weight, _, _, ldw = _as_matrix(weight)
        _one_device("blockwise_mm", x2, weight, bias)
        bias = _dense_bias(bias, n, x.dtype)
        xr, xc, w = N.BlockForm(m, k, "row"), N.BlockForm(m, k, "col"), N.BlockForm(n, k, "square")
        kept = torch.empty(w.nbytes + (xc.nbytes if need_dw else 0), dtype=torch.uint8, device=x.device)
        passing = torch.empty(xr.nbytes + N.GEMM_WORKSPACE_BYTES, dtype=torch.uint8, device=x.device)
        w.at(kept.data_ptr())
        if need_dw:
            xc.at(kept.data_ptr() + w.nbytes)
        xr.at(passing.data_ptr())
        N.block_cast_into(x2, ldx, xr, xc if need_dw else None)
        N.block_cast_into(weight, ldw, w, None)
        y = torch.empty((m, n), dtype=x.dtype, device=x.device)
        N.block_gemm_into(xr.operand(), w.operand(), bias, y, m, n, k, passing.data_ptr() + xr.nbytes)
        ctx.save_for_backward(kept)
        ctx.forms = (w, xc if need_dw else None)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], n)

    @staticmethod
    def _backward_eager(ctx, go, go2, need_dx, need_dw):
        (kept,), (w, xc) = ctx.saved_tensors, ctx.forms
        if kept.data_ptr() != w.data:  # packed away and unpacked elsewhere meanwhile
            moved = kept.data_ptr() - w.data
            w = N.BlockForm(w.rows, w.cols, "square").at(w.data + moved)
            xc = xc and N.BlockForm(xc.rows, xc.cols, "col").at(xc.data + moved)
        (m, n), k = go2.shape, w.cols
        go2, _, _, ldg = _as_matrix(go2)
        _one_device("blockwise_mm", kept, go2)
        gr, gc = N.BlockForm(m, n, "row") if need_dx else None, N.BlockForm(m, n, "col") if need_dw else None
        sizes = [f.nbytes if f else 0 for f in (gr, gc)]
        buf = torch.empty(sum(sizes) + 2 * N.GEMM_WORKSPACE_BYTES, dtype=torch.uint8, device=go.device)
        at = buf.data_ptr()
        if need_dx:
            gr.at(at)
        if need_dw:
            gc.at(at + sizes[0])
        ws = at + sum(sizes)
        N.block_cast_into(go2, ldg, gr, gc)
        dx = dw = None
        if need_dx:  # dX = dY @ W: the weight's bytes and factors read transposed
            dx = torch.empty((m, k), dtype=go.dtype, device=go.device)
            N.block_gemm_into(gr.operand(), w.operand(transposed=True), None, dx, m, k, n, ws)
            dx = dx if go.dim() == 2 else dx.reshape(*go.shape[:-1], k)
        if need_dw:  # dW = dY^T @ X, summed over rows: both by columns
            dw = torch.empty((n, k), dtype=ctx.dtypes[0], device=go.device)
            N.block_gemm_into(gc.operand(transposed=True), xc.operand(transposed=True), None, dw, n, k, m,
                              ws + N.GEMM_WORKSPACE_BYTES)
        return dx, dw

    @staticmethod
    def forward(ctx, x, weight, bias, need_dw: bool):
        x2 = x.reshape(-1, x.shape[-1])
        ctx.dtypes = (weight.dtype, bias.dtype if bias is not None else None)
        ctx.forms = None
        if x2.shape[1] != weight.shape[1]:
            raise RuntimeError(f"blockwise linear: the input has {x2.shape[1]} features, the weight {weight.shape[1]}")
        if eager_cuda(x) and eager_cuda(weight) and x2.numel() and weight.numel():
            return _float8_linear_blockwise._forward_eager(ctx, x, x2, weight, bias, need_dw)
        (x8, sx, ex), by_col = _cast(x2, N.E4M3, True, need_dw)
        w8, sw, ew, ewt = _cast_square(weight, N.E4M3)
        y = _mm(x8, w8, sx, sw, 1, BLOCK, ex, ew, bias, x.dtype)
        ctx.save_for_backward(*by_col, w8, sw, ewt)
        return y.reshape(*x.shape[:-1], y.shape[-1])

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        need_dx, need_dw, need_db = ctx.needs_input_grad[:3]
        go2 = go.reshape(-1, go.shape[-1])
        dx = dw = db = None
        if ctx.forms is not None and eager_cuda(go):
            if need_dx or need_dw:
                dx, dw = _float8_linear_blockwise._backward_eager(ctx, go, go2, need_dx, need_dw)
            if need_db:
                db = go2.sum(0, dtype=torch.float32).to(ctx.dtypes[1])
            return dx, dw, db, None
        if ctx.forms is not None:  # an eager forward whose backward is traced or watched
            (kept,), (w, xc) = ctx.saved_tensors, ctx.forms
            x8c, sxc, exc = xc.tensors(kept, w.nbytes) if xc is not None else (None, None, None)
            w8, sw, ewt = w.tensors(kept, 0)
        else:
            x8c, sxc, exc, w8, sw, ewt = ctx.saved_tensors
        if need_dx or need_dw:
            (g8, sg, eg), (g8c, sgc, egc) = _cast(go2, N.E4M3, need_dx, need_dw)
        if need_dx:  # dX = dY @ W: the weight's bytes and factors read transposed
            dx = _mm(g8, w8.t(), sg, sw.t(), 1, BLOCK, eg, ewt, None, go.dtype)
            dx = dx.reshape(*go.shape[:-1], dx.shape[-1])
        if need_dw:  # dW = dY^T @ X, summed over rows: both by columns
            dw = _mm(g8c.t(), x8c.t(), sgc.t(), sxc.t(), 1, 1, egc, exc, None, ctx.dtypes[0])
        if need_db:
            db = go2.sum(0, dtype=torch.float32).to(ctx.dtypes[1])
        return dx, dw, db, None
