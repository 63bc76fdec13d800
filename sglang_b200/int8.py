"""Weight-side objects of the W8A8 int8 path: the quantisation config and the linear "quant method" that create the parameters
of a checkpoint with int8 weights and one scale per output channel, and call the operators.

The parameters are ``weight`` int8 ``[N, K]`` and ``weight_scale`` fp32 ``[N, 1]``, the names that such checkpoints use, so that a
state dict loads as is. Dynamic symmetric activations only; expert weights are not built.
"""
from __future__ import annotations

from typing import Any, Dict, List, Optional, Tuple, Union

import torch

from .int8_kernel import int8_scaled_mm, w8a8_int8_linear


class W8A8Int8Config:
    """``quantization_config`` of a W8A8 int8 checkpoint."""

    def __init__(self, ignored_layers: Optional[List[str]] = None):
        self.ignored_layers = ignored_layers or []

    def get_name(self) -> str:
        return "w8a8_int8"

    @classmethod
    def from_config(cls, config: Dict[str, Any]) -> "W8A8Int8Config":
        if config.get("is_dynamic") is False:
            raise NotImplementedError("static activation scales are not built")
        return cls(ignored_layers=config.get("ignore", config.get("modules_to_not_convert")))

    def is_layer_skipped(self, prefix: str) -> bool:
        return any(prefix == name or prefix.startswith(name + ".") for name in self.ignored_layers)


class W8A8Int8LinearMethod:
    """Creates ``weight`` / ``weight_scale`` on a layer and applies the int8 linear."""

    def __init__(self, quant_config: W8A8Int8Config):
        self.quant_config = quant_config

    def create_weights(self, layer: torch.nn.Module, input_size_per_partition: int, output_partition_sizes: List[int],
                       input_size: int, output_size: int, params_dtype: torch.dtype, device=None, **extra) -> None:
        out_per_part = sum(output_partition_sizes)
        layer.logical_widths = list(output_partition_sizes)
        layer.input_size_per_partition = input_size_per_partition
        layer.output_size_per_partition = out_per_part
        layer.orig_dtype = params_dtype
        weight = torch.empty(out_per_part, input_size_per_partition, dtype=torch.int8, device=device)
        layer.register_parameter("weight", torch.nn.Parameter(weight, requires_grad=False))
        scale = torch.full((out_per_part, 1), torch.finfo(torch.float32).min, dtype=torch.float32, device=device)
        layer.register_parameter("weight_scale", torch.nn.Parameter(scale, requires_grad=False))

    def process_weights_after_loading(self, layer: torch.nn.Module) -> None:
        assert layer.weight.dtype == torch.int8, "weight is not int8"
        assert torch.all(layer.weight_scale.data > torch.finfo(torch.float32).min), "weight_scale not loaded"
        layer.weight = torch.nn.Parameter(layer.weight.data.contiguous(), requires_grad=False)
        layer.weight_scale = torch.nn.Parameter(layer.weight_scale.data.float().contiguous(), requires_grad=False)

    def apply(self, layer: torch.nn.Module, x: Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]],
              bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``x`` is the 16-bit activation, or what ``rmsnorm_quant_int8`` and ``per_token_quant_int8`` made of it:
        ``(x_q, x_s)``; the result is then of the type the layer was created for."""
        if isinstance(x, tuple):
            x_q, x_s = x[:2]
            out = int8_scaled_mm(x_q.reshape(-1, x_q.shape[-1]), layer.weight.t(), x_s, layer.weight_scale, layer.orig_dtype, bias)
            return out.view(*x_q.shape[:-1], out.shape[-1])
        return w8a8_int8_linear(x, layer.weight, layer.weight_scale, bias)


def quant_weight_int8(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """A 16-bit or fp32 weight ``[N, K]`` as int8 with one scale per output channel ``[N, 1]``: how such checkpoints are made
    (amax / 127 per row, nearest integer). On the device of the weight."""
    assert weight.dim() == 2, "weight must be a 2D tensor"
    w = weight.float()
    scale = w.abs().amax(-1, keepdim=True).clamp_min(1e-10) / torch.full((), 127.0, device=w.device)
    return (w / scale).round().clamp(-127, 127).to(torch.int8), scale
