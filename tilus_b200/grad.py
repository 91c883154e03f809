"""Which calls autograd follows, and what becomes of it at operators that have no backward pass."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad


def followed(*operands) -> bool:
    """Whether autograd is to record a call with these operands (tensors or None), backward or forward."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands):
        return True
    # (a dual tensor need not require a gradient; unpack_dual is asked only where forward mode is on)
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in operands)


class _NoBackward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, name, call):
        ctx.name = name
        return call(x)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no gradient with respect to its activations: detach() them where a backward pass is to "
                           "end, or run under torch.no_grad()")


def without_backward(name: str, call, x: torch.Tensor) -> torch.Tensor:
    """call(x), whose result refuses a backward pass instead of ending it in silence."""
    return _NoBackward.apply(x, name, call)
