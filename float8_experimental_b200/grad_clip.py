"""Norm of all gradients as one vector, and clipping to it: `torch.nn.utils.clip_grad_norm_` in three launches
(partial sums of every tensor, their sum, the scaling, which the device skips when nothing exceeds the bound) in
place of several per tensor, and without a host synchronisation.

Gradients of one call lie on one device; bf16, fp16 and fp32 may be mixed.  Clipping refuses gradients that overlap in
memory, except for one gradient tensor under several parameters, which counts and is scaled once.  DTensor
gradients (FSDP2, tensor parallel) count once over their mesh: the local sums are all-reduced over the mesh
dimensions a tensor is sharded on.
"""
from __future__ import annotations

import math
from typing import Dict, Iterable, List, Union

import torch
import torch.distributed as dist
from torch.autograd.graph import increment_version
from torch.distributed._tensor import DTensor

from . import _native as N
from ._ops import _PLAIN as _PLAIN_TYPES, eager_cuda, ops, TensorList

__all__ = ["get_total_norm", "clip_grads_with_norm_", "clip_grad_norm_"]

_PLAIN = set(_PLAIN_TYPES)
_KINDS = {math.inf: 0, 1.0: 1, 2.0: 2}


def _kind_of(norm_type: float) -> int:
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type}")
    return kind


def _local(t: torch.Tensor) -> torch.Tensor:
    return t._local_tensor if isinstance(t, DTensor) else t


def _gradients(parameters: Union[torch.Tensor, Iterable[torch.Tensor]]) -> List[torch.Tensor]:
    """The gradients of `parameters`, each once however often it or its parameter is listed."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [g for p in params if (g := p.grad) is not None]
    if len(set(map(id, grads))) != len(grads):  # a parameter listed twice, or parameters that share one gradient tensor
        grads = list({id(g): g for g in grads}.values())
    return grads


def _sharded_groups(t: DTensor):
    """The process groups whose ranks hold different parts of `t`."""
    groups = []
    for dim, placement in enumerate(t.placements):
        if placement.is_partial():
            raise NotImplementedError("gradient norm of a Partial DTensor")
        if not placement.is_replicate():  # Shard, or FSDP2's strided shard on top of a tensor-parallel one: no Shard by its type
            groups.append(t.device_mesh.get_group(dim))
    return tuple(groups)


def _total_norm(tensors: List[torch.Tensor], kind: int) -> torch.Tensor:
    if not tensors:
        return torch.tensor(0.0)
    if not any(isinstance(t, DTensor) for t in tensors):
        return ops.multi_norm(tensors, kind, True)
    by_groups: Dict[tuple, List[torch.Tensor]] = {}
    for t in tensors:
        by_groups.setdefault(_sharded_groups(t) if isinstance(t, DTensor) else (), []).append(_local(t))
    parts = []
    for groups, local in by_groups.items():
        part = ops.multi_norm(local, kind, False)
        for group in groups:
            dist.all_reduce(part, op=dist.ReduceOp.MAX if kind == 0 else dist.ReduceOp.SUM, group=group)
        parts.append(part)
    both = torch.stack(parts)
    return both.max() if kind == 0 else both.sum().sqrt() if kind == 2 else both.sum()


def _scale(grads: List[torch.Tensor], total: torch.Tensor, max_norm: float) -> None:
    ops.multi_clip_([_local(g) for g in grads], total, float(max_norm))
    wrappers = [g for g in grads if isinstance(g, DTensor)]
    if wrappers:  # the operator has seen to the versions of what it was given
        increment_version(wrappers)


def _check_finite(total: torch.Tensor, norm_type: float) -> None:
    if not bool(torch.isfinite(total)):
        raise RuntimeError(
            f"The total norm of order {norm_type} for gradients is non-finite, so it cannot be clipped. "
            "To disable this error and scale the gradients by the non-finite norm anyway, set `error_if_nonfinite=False`"
        )


@torch.no_grad()
def get_total_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0,
                   error_if_nonfinite: bool = False) -> torch.Tensor:
    """The `norm_type` (1, 2 or inf) norm of all `tensors` together, fp32, 0-dim, on their device.  No tensors: 0.
    A tensor that is listed twice counts twice (the functions that take parameters count each gradient once).

    Squares are formed in fp32 as in torch: an element beyond 1.8e19 makes the 2-norm infinite."""
    kind = _kind_of(norm_type)
    total = _total_norm([tensors] if isinstance(tensors, torch.Tensor) else list(tensors), kind)
    if error_if_nonfinite:
        _check_finite(total, norm_type)
    return total


@torch.no_grad()
def clip_grads_with_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float,
                          total_norm: torch.Tensor) -> None:
    """Multiplies every gradient by min(1, max_norm / (total_norm + 1e-6)), in place.  A NaN norm makes them NaN."""
    grads = _gradients(parameters)
    if grads:
        _scale(grads, total_norm, max_norm)


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clips the gradients of `parameters` to a total norm of at most `max_norm`, in place, and returns the norm they had
    (fp32, 0-dim, on their device).  `error_if_nonfinite=True` reads it back and synchronises."""
    kind = _kind_of(norm_type)
    grads = _gradients(parameters)
    if grads and set(map(type, grads)) <= _PLAIN and eager_cuda(grads[0]):
        # the usual case: the tensors' addresses are gathered once for both launches
        tensors = TensorList("clip_grad_norm_", grads)
        total = torch.empty((), dtype=torch.float32, device=tensors.device)
        N.multi_norm(tensors, kind, True, total)
        if error_if_nonfinite:
            _check_finite(total, norm_type)
        N.multi_clip(tensors, total, float(max_norm))
        increment_version(grads)  # a backward pass that still needs one of them must not take the scaled values for it
        return total
    total = _total_norm(grads, kind)
    if error_if_nonfinite:
        _check_finite(total, norm_type)
    if grads:
        _scale(grads, total, max_norm)
    return total
