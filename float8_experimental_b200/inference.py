"""Float8 inference linear: weight quantised once, activations cast per call, the product
on the tcgen05 GEMM with the bias fused into its epilogue
(API of float8_experimental/inference.py:30-244).
"""
from __future__ import annotations

from dataclasses import dataclass
from enum import auto, Enum
from typing import Callable, Optional

import torch
import torch.nn as nn

from .float8_blockwise import BLOCK, cast_to_float8_blockwise, linear_by_rows
from .float8_linear_utils import swap_linear_layers
from .float8_tensor import (
    Float8Tensor,
    GemmInputRole,
    hp_tensor_and_scale_to_float8,
    LinearMMConfig,
    ScaledMMConfig,
    tensor_already_casted_to_fp8,
)
from .float8_utils import e4m3_dtype, tensor_to_scale


class ActivationCasting(Enum):
    """How activations reach the GEMM (reference: inference.py:30-42).

    WEIGHT_ONLY  weights stored in fp8, dequantised for a high-precision matmul
    DYNAMIC      activations cast per call with a scale from their own amax
    STATIC       activations cast per call with a fixed, calibrated scale
    BLOCKWISE    activations cast per call with a scale per row and 128 columns, weights with one per 128 x 128
                 square: `weight` holds the fp8 bytes, the buffer `weight_scale_inv` the squares' factors (any
                 fp32 values, so a checkpoint that brings both can be loaded into them)"""

    WEIGHT_ONLY = auto()
    DYNAMIC = auto()
    STATIC = auto()
    BLOCKWISE = auto()


@dataclass(frozen=True)
class QuantConfig:
    """Quantisation recipe of an inference linear (reference: inference.py:45-66)."""

    activation_casting: ActivationCasting
    static_quantization_scale: Optional[torch.Tensor] = None
    # class attribute, as in the reference: zero-pad the inner GEMM dimension to 16
    pad_inner_dim = False

    def __post_init__(self):
        if self.activation_casting == ActivationCasting.STATIC:
            assert isinstance(
                self.static_quantization_scale, torch.Tensor
            ), "When activation_casting is 'static', activation_scale must be a tensor."


def cast_to_float8_e4m3_inference(
    inpt_tensor: torch.Tensor,
    linear_mm_config: LinearMMConfig,
    reduce_amax: bool = False,
    static_quantization_scale: Optional[torch.Tensor] = None,
) -> Float8Tensor:
    """Activation -> e4m3 `Float8Tensor`, with the static scale when one is given, else a
    dynamic one; already-fp8 inputs pass through (reference: inference.py:179-211)."""
    if tensor_already_casted_to_fp8(inpt_tensor):
        return inpt_tensor
    scale = static_quantization_scale
    if scale is None:
        scale = tensor_to_scale(inpt_tensor, e4m3_dtype, reduce_amax)
    return hp_tensor_and_scale_to_float8(
        inpt_tensor, scale, e4m3_dtype, linear_mm_config, GemmInputRole.INPUT, with_transpose=False
    )


class Float8InferenceLinear(torch.nn.Linear):
    """`nn.Linear` for inference with an fp8 weight (reference: inference.py:69-176)."""

    def __init__(self, quant_config: QuantConfig, linear_mm_config: LinearMMConfig, in_features: int,
                 out_features: int, bias: bool = True, device: Optional[torch.device] = None,
                 dtype: Optional[torch.dtype] = None) -> None:
        super().__init__(in_features, out_features, bias, device, dtype)
        self.linear_mm_config = linear_mm_config
        self.activation_casting = quant_config.activation_casting
        if self.activation_casting == ActivationCasting.STATIC:
            self.register_buffer("static_quantization_scale", quant_config.static_quantization_scale)
        else:
            self.static_quantization_scale = None

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        if self.activation_casting == ActivationCasting.BLOCKWISE:
            return self._forward_blockwise(input)
        if self.activation_casting == ActivationCasting.WEIGHT_ONLY:
            return torch.nn.functional.linear(input, self.weight.to_original_precision())
        x_fp8 = cast_to_float8_e4m3_inference(
            input, self.linear_mm_config, static_quantization_scale=self.static_quantization_scale
        )
        # linear(Float8Tensor, Float8Tensor, bias) lands in the op table's mm / addmm
        return torch.nn.functional.linear(x_fp8, self.weight, self.bias)

    def _forward_blockwise(self, input: torch.Tensor) -> torch.Tensor:
        if tensor_already_casted_to_fp8(input):
            raise RuntimeError(f"ActivationCasting.BLOCKWISE takes plain tensors, got a {type(input).__name__}")
        return linear_by_rows(input, self.weight, self.weight_scale_inv, self.bias)

    def quantize_weight(self, dtype: torch.dtype = e4m3_dtype) -> None:
        """Replaces the weight by its `Float8Tensor` (dynamic scale), frozen; with ActivationCasting.BLOCKWISE by its
        fp8 bytes and the buffer `weight_scale_inv`."""
        assert not isinstance(self.weight, Float8Tensor) and self.weight.element_size() > 1, \
            "Weight has already been quantized, cannot quantize again."
        if self.activation_casting == ActivationCasting.BLOCKWISE:
            w8 = cast_to_float8_blockwise(self.weight, (BLOCK, BLOCK), dtype)
            self.weight = nn.Parameter(w8.data, requires_grad=False)
            self.register_buffer("weight_scale_inv", w8.scale_inv)
            return
        with torch.no_grad():
            scale = tensor_to_scale(self.weight, dtype)
            w8 = hp_tensor_and_scale_to_float8(
                self.weight, scale, dtype, self.linear_mm_config, GemmInputRole.WEIGHT, with_transpose=False
            )
        self.weight = nn.Parameter(w8)
        self.weight.requires_grad = False

    def set_weight_and_bias(self, weight: torch.nn.Parameter, bias: Optional[torch.nn.Parameter]):
        self.weight = weight
        self.bias = bias

    @classmethod
    def from_float(cls, module: nn.Module, quant_config: QuantConfig, use_fast_accum: bool) -> "Float8InferenceLinear":
        """Builds the inference linear from an `nn.Linear`, sharing then quantising its weight."""
        fwd = ScaledMMConfig(False, use_fast_accum, pad_inner_dim=quant_config.pad_inner_dim)
        linear = cls(quant_config, LinearMMConfig(fwd, fwd, fwd), module.in_features, module.out_features, False,
                     device=torch.device("meta"))
        linear.set_weight_and_bias(module.weight, module.bias)
        linear.quantize_weight()
        return linear


def quantize_to_float8(
    module: nn.Module,
    quant_config: QuantConfig,
    *,
    module_filter_fn: Optional[Callable[[nn.Module, str], bool]] = None,
    use_fast_accum: bool = True,
) -> nn.Module:
    """Swaps `nn.Linear` for `Float8InferenceLinear` throughout `module`
    (reference: inference.py:214-244)."""
    return swap_linear_layers(
        module,
        lambda m: Float8InferenceLinear.from_float(m, quant_config, use_fast_accum),
        module_filter_fn=module_filter_fn,
    )
