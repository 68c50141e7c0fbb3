"""Layer norm and root-mean-square norm of an expert layer's rows, with the residual added first, and their gradients.

    entered = rms_norm(attention, gamma, residual=h)      # entered.residual = attention + h, entered.normalized = its norm
    logits = entered.normalized.float() @ router.T
    ...
    h = combine_weighted(y, handle.token_slots, weights, bias=entered.residual)

`rms_norm_fp8` is the one for serving in 8 bits; these two are in bf16 or fp32, for training and for serving without 8 bits, and
autograd finds their gradients.  The two `_backward` calls are those gradients, for callers that do without autograd.

Calls run on the caller's current stream; nothing is copied to the host.  `ValueError` for misuse of arguments, as `Buffer` has it;
`RuntimeError` where a derivative is asked for that an operator does not have: in forward mode, or of a gradient.
Calls can be captured into a graph, and so can autograd's backward pass, as long as no eager result of the same leaves is kept
meanwhile: autograd would wait for its stream.
None of this has a counterpart in the reference.
"""

from __future__ import annotations

import dataclasses
from typing import Optional

import torch

from ._native import load_extension
from .operators import _dense

__all__ = ["NormResult", "layer_norm", "layer_norm_backward", "rms_norm", "rms_norm_backward"]


@dataclasses.dataclass
class NormResult:
    """normalized: the norm; residual: x + residual, which is what was normed, None without one; mean (None of a root-mean-square
    norm) and rstd: fp32 [tokens], as the `_backward` calls take them."""

    normalized: torch.Tensor
    residual: Optional[torch.Tensor]
    mean: Optional[torch.Tensor]
    rstd: torch.Tensor


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, residual, eps, centred):
        ctx.set_materialize_grads(False)
        extension = load_extension()
        if centred:
            normalized, total, mean, rstd = extension.layer_norm(x, gamma, beta, residual, eps)
        else:
            normalized, total, mean, rstd = extension.rms_norm(x, gamma, residual, eps)
        ctx.save_for_backward(x if total is None else total, gamma, mean, rstd)
        ctx.mark_non_differentiable(*(tensor for tensor in (mean, rstd) if tensor is not None))
        return normalized, total, mean, rstd

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, grad_residual, _mean, _rstd):
        total, gamma, mean, rstd = ctx.saved_tensors
        needs_x, needs_gamma, needs_beta, needs_residual = ctx.needs_input_grad[:4]
        if grad is None:  # only the sum was used
            return grad_residual if needs_x else None, None, None, grad_residual if needs_residual else None, None, None
        grad = _dense(grad)
        grad_residual = None if grad_residual is None else _dense(grad_residual)
        wanted = {"input": needs_x or needs_residual, "parameters": needs_gamma or needs_beta}
        if mean is None:
            grad_x, grad_gamma = rms_norm_backward(grad, total, gamma, rstd, grad_residual=grad_residual, **wanted)
            grad_beta = None
        else:
            grad_x, grad_gamma, grad_beta = layer_norm_backward(grad, total, gamma, mean, rstd, grad_residual=grad_residual, **wanted)
        return (grad_x if needs_x else None, grad_gamma if needs_gamma else None, grad_beta if needs_beta else None,
                grad_x if needs_residual else None, None, None)


def _tracked(*tensors) -> bool:
    return torch.is_grad_enabled() and any(tensor is not None and tensor.requires_grad for tensor in tensors)


def layer_norm(
    x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor | None = None, *, residual: torch.Tensor | None = None, eps: float = 1e-5
) -> NormResult:
    """s = x + residual, rounded to x's type; (s - mean(s)) / sqrt(mean((s - mean(s))^2) + eps) * gamma + beta, in fp32 and rounded
    once.  x and residual: contiguous bf16 or fp32 [tokens, hidden]; gamma and beta: [hidden] of x's type or fp32, both the same;
    hidden a multiple of 8 up to 16384.

    It has a gradient in x, residual, gamma and beta; sums over the rows are in fp32 and in the same order every time."""
    if _tracked(x, gamma, beta, residual):
        return NormResult(*_Norm.apply(x, gamma, beta, residual, eps, True))
    return NormResult(*load_extension().layer_norm(x, gamma, beta, residual, eps))


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6) -> NormResult:
    """s = x + residual, rounded to x's type; s / sqrt(mean(s^2) + eps) * gamma, in fp32 and rounded once.  Arguments and gradients
    as `layer_norm` has them."""
    if _tracked(x, gamma, residual):
        return NormResult(*_Norm.apply(x, gamma, None, residual, eps, False))
    return NormResult(*load_extension().rms_norm(x, gamma, residual, eps))


def layer_norm_backward(
    grad: torch.Tensor,
    total: torch.Tensor,
    gamma: torch.Tensor,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    *,
    grad_residual: torch.Tensor | None = None,
    input: bool = True,
    parameters: bool = True,
) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """The gradients (grad_x, which is residual's as well; grad_gamma; grad_beta) of `layer_norm` for the gradient of its `normalized`
    and, with `grad_residual`, of its `residual`.  total: the rows that were normed (x, or with a residual the result's
    `residual`).  Without `input`, grad_x is None; without `parameters`, the other two.  Without a gradient of its own."""
    return load_extension().layer_norm_backward(grad, total, gamma, mean, rstd, grad_residual, input, parameters)


def rms_norm_backward(
    grad: torch.Tensor,
    total: torch.Tensor,
    gamma: torch.Tensor,
    rstd: torch.Tensor,
    *,
    grad_residual: torch.Tensor | None = None,
    input: bool = True,
    parameters: bool = True,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """The gradients (grad_x, grad_gamma) of `rms_norm`, as `layer_norm_backward` has them."""
    return load_extension().rms_norm_backward(grad, total, gamma, rstd, grad_residual, input, parameters)[:2]
