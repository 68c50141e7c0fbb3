"""The router of an expert layer: which experts a token goes to and with what weights, the loss that balances the experts, and the
gradients of both.

    routing = route_topk(logits, 8, scoring="sigmoid", bias=bias, groups=8, topk_groups=4, scale=2.5)
    received = buffer.dispatch(x, topk_idx=routing.ids, do_expand=True)
    out = combine_weighted(y, received.handle.token_slots, routing.weights)
    balance = balance_loss(logits, routing.ids, scoring="sigmoid")         # balance.loss, and the choices of every expert
    bias += step * (balance.counts.float().mean() - balance.counts).sign()

A score is a token's softmax over the experts, or the sigmoid of each logit.

Calls run on the caller's current stream; nothing is copied to the host.  `ValueError` for misuse of arguments, as `Buffer` has it;
`RuntimeError` where a derivative is asked for that an operator does not have: in forward mode, or of a gradient.
Calls can be captured into a graph, and so can autograd's backward pass, as long as no eager result of the same leaves is kept
meanwhile: autograd would wait for its stream.
None of this has a counterpart in the reference, whose routing is the caller's.
"""

from __future__ import annotations

import dataclasses

import torch

from ._native import load_extension

__all__ = ["BalanceResult", "Routing", "balance_loss", "balance_loss_backward", "route_topk", "route_topk_backward"]

_SCORINGS = {"softmax": 0, "sigmoid": 1}


def _scoring(name: str) -> int:
    if name not in _SCORINGS:
        raise ValueError(f"scoring must be one of {', '.join(_SCORINGS)}")
    return _SCORINGS[name]


@dataclasses.dataclass
class Routing:
    """ids: int64 [tokens, topk], as `Buffer.dispatch` takes them, -1 where masked; weights: float32 [tokens, topk], zero there."""

    ids: torch.Tensor
    weights: torch.Tensor


@dataclasses.dataclass
class BalanceResult:
    """loss: float32 [] or, with sequences, [sequences]; counts: int64 [experts] or [sequences, experts], every expert's choices;
    tokens: int64 [] or [sequences], the tokens that have a choice."""

    loss: torch.Tensor
    counts: torch.Tensor
    tokens: torch.Tensor


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, scoring, bias, mask, groups, topk_groups, normalize, scale):
        ctx.set_materialize_grads(False)
        ids, weights = load_extension().route_topk(logits, topk, scoring, bias, mask, groups, topk_groups, normalize, scale)
        ctx.save_for_backward(logits, ids)
        ctx.mark_non_differentiable(ids)
        ctx.scores = (scoring, normalize, scale)
        return ids, weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _ids, grad):
        logits, ids = ctx.saved_tensors
        found = None if grad is None else load_extension().route_topk_backward(grad.contiguous(), logits, ids, *ctx.scores)
        return found, None, None, None, None, None, None, None, None


def route_topk(
    logits: torch.Tensor,
    topk: int,
    *,
    scoring: str = "softmax",
    bias: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    groups: int = 1,
    topk_groups: int = 1,
    normalize: bool = True,
    scale: float = 1.0,
) -> Routing:
    """Every token's `topk` experts of the largest value, in descending order, the lowest index first among equals, and their weights:
    scale times the chosen experts' scores, with `normalize` divided by the chosen ones' sum, in fp32.

    An expert's value is its logit, the order of its score; with `bias` (float32 [experts]) or groups it is its score, plus the bias,
    in 64 bits, so that neither the order of a sum nor an exponential's last bit decides.  The bias is in no weight and has no
    gradient.  With `topk_groups` < `groups`, the experts fall into groups of neighbours, a group is as good as the sum of its two
    largest values (also without a bias), and only the `topk_groups` best groups are chosen from.

    logits: bf16 or fp32 [tokens, experts], up to 4096 experts, rows any distance apart; topk up to 32.  An expert whose logit (or
    value) is -infinity is never chosen; choices that find no expert are -1 with weight 0, and so are all choices of tokens whose
    `mask` (bool [tokens]) is False, whose logits are not looked at.  NaN is above everything; ids stay distinct.  A NaN makes all of its
    token's weights NaN, and so does an infinite logit in a softmax; of sigmoids without `normalize` only the NaN's own weight is.
    The weights have a gradient in the logits."""
    arguments = (logits, topk, _scoring(scoring), bias, mask, groups, topk_groups, normalize, scale)
    if logits.requires_grad and torch.is_grad_enabled():
        return Routing(*_Route.apply(*arguments))
    return Routing(*load_extension().route_topk(*arguments))


def route_topk_backward(
    grad: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, *, scoring: str = "softmax", normalize: bool = True, scale: float = 1.0
) -> torch.Tensor:
    """The gradient [tokens, experts] in the logits of `route_topk`'s weights, for their gradient (float32 [tokens, topk]), in the
    logits' type.  An id outside the experts is a masked choice; one that a token has twice counts twice.  Without a gradient of its own."""
    return load_extension().route_topk_backward(grad, logits, ids, _scoring(scoring), normalize, scale)


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, scoring, sequence_offsets):
        ctx.set_materialize_grads(False)
        loss, counts, tokens = load_extension().balance_loss(logits, ids, scoring, sequence_offsets)
        # (copies: a user adds up counts in place, over ranks with a collective that autograd does not see)
        ctx.save_for_backward(logits, ids, counts.clone(), tokens.clone(), sequence_offsets)
        ctx.mark_non_differentiable(counts, tokens)
        ctx.scoring = scoring
        return loss, counts, tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _counts, _tokens):
        if grad is None:
            return None, None, None, None
        logits, ids, counts, tokens, sequence_offsets = ctx.saved_tensors
        found = load_extension().balance_loss_backward(grad.contiguous(), logits, ids, counts, tokens, ctx.scoring, sequence_offsets)
        return found, None, None, None


def balance_loss(
    logits: torch.Tensor, ids: torch.Tensor, *, scoring: str = "softmax", sequence_offsets: torch.Tensor | None = None
) -> BalanceResult:
    """How evenly a batch's choices fall on the experts: experts * sum over e of counts[e] / (all choices) * the mean of e's share over
    the tokens.  A share is the softmax of the token's logits, or its sigmoid over the sum of them; the loss is 1 where either the
    choices or the shares are even, and grows with experts that are both chosen and scored more often.

    ids: int64 [tokens, topk], as `route_topk` gives them; ids outside the experts are masked choices.  A token without a choice is
    padding: its logits are not looked at, its gradient is zero.  With `sequence_offsets` (int64 [sequences + 1], from 0 on, ascending)
    each sequence [offsets[s], offsets[s + 1]) has a loss, counts and tokens of its own; tokens behind the last one are none's.  A
    sequence without a choice has the loss 0.  The loss has a gradient in the logits, in which the counts are constants; the result's
    `counts` and `tokens` may be changed or reduced in place ahead of the backward pass."""
    arguments = (logits, ids, _scoring(scoring), sequence_offsets)
    if logits.requires_grad and torch.is_grad_enabled():
        return BalanceResult(*_BalanceLoss.apply(*arguments))
    return BalanceResult(*load_extension().balance_loss(*arguments))


def balance_loss_backward(
    grad: torch.Tensor,
    logits: torch.Tensor,
    ids: torch.Tensor,
    counts: torch.Tensor,
    tokens: torch.Tensor,
    *,
    scoring: str = "softmax",
    sequence_offsets: torch.Tensor | None = None,
) -> torch.Tensor:
    """The gradient [tokens, experts] of `balance_loss` in the logits, in their type, for the loss's gradient and the counts and tokens
    that the loss came with.  Without a gradient of its own."""
    return load_extension().balance_loss_backward(grad, logits, ids, counts, tokens, _scoring(scoring), sequence_offsets)
