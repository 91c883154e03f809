"""BlockNorm: the norms before and after a decoder block with its gate and residual scale, as a module.

ops.block_norm and ops.block_norm_backward are the operators; this module holds their weights and ties them together for
autograd.  The layers of this package have no backward pass: gradients come as far as the norms that no such layer stands behind.
"""
from __future__ import annotations

import torch
from torch import nn

from . import ops
from .dtypes import act_dtype
from .grad import followed

_TORCH_ACT = {"float16": torch.float16, "bfloat16": torch.bfloat16}


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, block, residual, weight, post_weight, gate, residual_scale, eps):
        ctx.save_for_backward(block, residual, weight, post_weight, gate)
        ctx.numbers = dict(residual_scale=residual_scale, eps=eps)
        ctx.set_materialize_grads(False)
        return ops.block_norm(block, residual, weight, post_weight=post_weight, gate=gate, **ctx.numbers)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_x, grad_new):
        block, residual, weight, post_weight, gate = ctx.saved_tensors
        if grad_x is None and grad_new is None:
            return (None,) * 7
        grad_x = torch.zeros_like(block) if grad_x is None else _rows(grad_x)
        got = ops.block_norm_backward(grad_x, None if grad_new is None else _rows(grad_new), block, residual, weight,
                                      post_weight=post_weight, gate=gate, **ctx.numbers)
        grads = [g if g is None else g.to(like.dtype)
                 for g, like in zip(got, (block, residual, weight, post_weight, gate))]
        return (*grads, None, None)


def _rows(grad: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernels take it: autograd hands over expanded and transposed ones too."""
    ok = grad.stride(1) == 1 and grad.stride(0) >= grad.shape[1] and grad.stride(0) % 8 == 0 and grad.data_ptr() % 16 == 0
    return grad if ok else grad.clone(memory_format=torch.contiguous_format)


def block_norm(block, residual, weight, *, post_weight=None, gate=None, residual_scale=1.0, eps=1e-6):
    """ops.block_norm as a function of torch's autograd (backward only; tangents are refused).  Not for stream capture while gradients
    are recorded: autograd's own bookkeeping outlives a capture; capture ops.block_norm and ops.block_norm_backward instead."""
    operands = (block, residual, weight, post_weight, gate)
    if followed(*operands):
        if block.is_cuda:
            with torch.cuda.device(block.device):
                capturing = torch.cuda.is_current_stream_capturing()
            if capturing:
                raise RuntimeError("block_norm records gradients and cannot be captured: capture ops.block_norm and "
                                   "ops.block_norm_backward, or capture under torch.no_grad()")
        return _BlockNorm.apply(*operands, residual_scale, eps)
    return ops.block_norm(block, residual, weight, post_weight=post_weight, gate=gate, residual_scale=residual_scale, eps=eps)


class BlockNorm(nn.Module):
    """Between two blocks: forward(block, residual) -> (x, new_residual), as ops.block_norm.

    ``post_norm``: the block's output is normed before it is added (post_weight).  ``gated``: a gate per channel (gate);
    forward() also takes one of its own, [gates, hidden], in its place.  Weights start at one and are of ``x_dtype``."""

    def __init__(self, x_dtype, hidden: int, post_norm: bool = False, gated: bool = False, residual_scale: float = 1.0,
                 eps: float = 1e-6):
        super().__init__()
        self.x_dtype = act_dtype(x_dtype)
        dtype = _TORCH_ACT[self.x_dtype.name]
        if hidden < 8 or hidden % 8 or hidden > 16384:
            raise ValueError("hidden must be a multiple of 8, at most 16384")
        self.hidden = hidden
        self.residual_scale = float(residual_scale)
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(hidden, dtype=dtype))
        self.post_weight = nn.Parameter(torch.ones(hidden, dtype=dtype)) if post_norm else None
        self.gate = nn.Parameter(torch.ones(hidden, dtype=dtype)) if gated else None

    def _operands(self, block, residual, gate):
        if block.dim() < 2 or block.shape[-1] != self.hidden:
            raise ValueError(f"expected rows of {self.hidden} channels")
        if residual is not None and residual.shape != block.shape:
            raise ValueError("residual must have the block's shape")
        rows = block.reshape(-1, self.hidden)
        return rows, None if residual is None else residual.reshape(-1, self.hidden), dict(
            post_weight=self.post_weight, gate=self.gate if gate is None else gate, residual_scale=self.residual_scale,
            eps=self.eps)

    def forward(self, block: torch.Tensor, residual: torch.Tensor | None, gate: torch.Tensor | None = None):
        rows, res, rest = self._operands(block, residual, gate)
        x, new = block_norm(rows, res, self.weight, **rest)
        return x.reshape(block.shape), new.reshape(block.shape)

    def forward_cast(self, block: torch.Tensor, residual: torch.Tensor | None, gate: torch.Tensor | None = None):
        """(x int8 [tokens, hidden], x_sf [tokens], new_residual) for Int8Linear.forward_cast; no gradients."""
        rows, res, rest = self._operands(block, residual, gate)
        x, sf, new = ops.block_norm_cast_int8(rows, res, self.weight, **rest)
        return x, sf, new.reshape(block.shape)

    def extra_repr(self) -> str:
        return (f"hidden={self.hidden}, x_dtype={self.x_dtype.name}, post_norm={self.post_weight is not None}, "
                f"gated={self.gate is not None}, residual_scale={self.residual_scale}, eps={self.eps}")
