"""Int8Linear: a linear layer in 8-bit integers on both sides, beside QuantizedLinear.

Where QuantizedLinear keeps 16-bit activations and is bound by reading its weights, this layer also casts the
activations (a scale per token) and multiplies at the integer rate of the tensor cores, twice the 16-bit one: for prompt
processing and large batches.  Weights are cast with a scale per output channel.
"""
from __future__ import annotations

import torch
from torch import nn

from . import ops
from .dtypes import act_dtype
from .grad import followed, without_backward

_TORCH_ACT = {"float16": torch.float16, "bfloat16": torch.bfloat16}


class Int8Linear(nn.Module):
    """Constructor arguments and loading as QuantizedLinear's, without a weight type and a group size:

        Int8Linear(x_dtype, in_features, out_features, bias=False)
          .weight : int8[out_features, in_features]
          .scales : float32[out_features]
          .bias   : x_dtype[out_features] or None

    in_features and out_features are multiples of 16.  The forward passes run the CUDA library; there is no CPU path.  They have
    no backward pass: where activations require a gradient, backward() through the result raises."""

    def __init__(self, x_dtype, in_features: int, out_features: int, bias: bool = False):
        super().__init__()
        self.x_dtype = act_dtype(x_dtype)
        self.act_torch_dtype = _TORCH_ACT[self.x_dtype.name]
        if in_features < 16 or out_features < 16 or in_features % 16 or out_features % 16:
            raise ValueError("in_features and out_features must be multiples of 16")
        self.in_features = in_features
        self.out_features = out_features
        self.weight = nn.Parameter(torch.zeros(out_features, in_features, dtype=torch.int8), requires_grad=False)
        self.scales = nn.Parameter(torch.ones(out_features, dtype=torch.float32), requires_grad=False)
        self.bias = nn.Parameter(torch.zeros(out_features, dtype=self.act_torch_dtype), requires_grad=False) if bias else None

    def _apply(self, fn, recurse=True):
        scales = self.scales.data
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:  # .half() and the like: the scales stay what they are
            self.scales.data = scales.to(self.scales.device)
        return self

    def load_and_quantize(self, weight: torch.Tensor, bias: torch.Tensor | None = None):
        """Cast a dense weight[out_features, in_features]: a scale per output channel.  A float32 weight is rounded to the
        activations' type first."""
        if tuple(weight.shape) != (self.out_features, self.in_features):
            raise ValueError(f"weight must be [{self.out_features}, {self.in_features}]")
        if (bias is None) != (self.bias is None):
            raise ValueError("a bias is given exactly where the layer has one")
        dev = self.weight.device
        w = weight.detach().to(device=dev)
        if w.dtype not in (torch.float16, torch.bfloat16):
            w = w.to(self.act_torch_dtype)
        if w.stride(1) != 1 or w.stride(0) % 8 or w.data_ptr() % 16:
            w = w.clone(memory_format=torch.contiguous_format)
        codes, scales = ops.per_token_cast_int8(w)
        with torch.no_grad():
            self.weight.copy_(codes)
            self.scales.copy_(scales)
            if bias is not None:
                self.bias.copy_(bias.to(dev))

    def _rows(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() == 0 or x.shape[-1] != self.in_features:
            raise ValueError(f"expected {self.in_features} input features")
        return x if x.dim() == 2 else x.reshape(-1, self.in_features)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x [..., in_features] in the activations' type: cast per token, then multiplied."""
        if followed(x):
            return without_backward("Int8Linear", self.forward, x)
        if x.dtype != self.act_torch_dtype:
            raise TypeError(f"activations must be {self.act_torch_dtype}")
        weight, rest = self.weight, dict(bias=self.bias, out_dtype=self.act_torch_dtype)
        # (early: the cast behind all that wrote the weights, which may be a parametrization just now, waits for it)
        codes, x_sf = ops.per_token_cast_int8(self._rows(x))
        out = ops.int8_matmul(codes, weight, x_sf, self.scales, early_b=True, **rest)
        return out if x.dim() == 2 else out.reshape(*x.shape[:-1], self.out_features)

    def forward_cast(self, x: torch.Tensor, x_sf: torch.Tensor, *, early_b: bool = False) -> torch.Tensor:
        """forward() for activations that are cast already (int8 [tokens, in_features], float32 [tokens]), by
        per_token_cast_int8 or block_norm_cast_int8.  ``early_b`` as for ops.int8_matmul: where that cast or norm stands
        directly in front and the weights (parameters, not computed on access) were written before it."""
        return ops.int8_matmul(x, self.weight, x_sf, self.scales, bias=self.bias, out_dtype=self.act_torch_dtype,
                               early_b=early_b)

    def forward_swiglu(self, x: torch.Tensor, x_sf: torch.Tensor | None = None, swiglu_clamp_value=None, *,
                       early_b: bool = False) -> torch.Tensor:
        """For a gate_up projection (out_features = 2 * hidden, gate rows first): silu(gate) * up [tokens, hidden] from one
        kernel.  ``x`` as forward() takes it, or with ``x_sf`` (and ``early_b``) as forward_cast() does."""
        if self.bias is not None:
            raise ValueError("a gate_up projection has no bias here")
        if followed(x):
            return without_backward("Int8Linear", lambda t: self.forward_swiglu(t, x_sf, swiglu_clamp_value, early_b=early_b), x)
        weight = self.weight
        if x_sf is None:
            if x.dtype != self.act_torch_dtype:
                raise TypeError(f"activations must be {self.act_torch_dtype}")
            x, x_sf = ops.per_token_cast_int8(self._rows(x))
            early_b = True  # as in forward()
        return ops.int8_gate_up(x, weight, x_sf, self.scales, out_dtype=self.act_torch_dtype,
                                swiglu_clamp_value=swiglu_clamp_value, early_b=early_b)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, x_dtype={self.x_dtype.name}, "
                f"bias={self.bias is not None}")
