"""The expert layer around `dispatch` and `combine`, in 8 bits: the norm ahead of it, the experts' two products, and
the combine that applies the gate weights, with its gradient.

    normed = rms_norm_fp8(x, gamma, residual=h, normalized=True)        # h + x, its norm in bf16 and in 8 bits
    received = buffer.dispatch(normed.rows.payload, topk_idx=idx, do_expand=True)     # 8-bit rows, moved as bf16
    layout = received.handle.layout
    rows = Fp8Rows.of_payload(received.x, hidden)
    act = experts_gated(rows, gate_up, layout.expert_offsets, layout.expert_counts)   # silu(gate) * up, in 8 bits
    y = experts_linear(act, down, layout.expert_offsets, layout.expert_counts)        # bf16
    out = combine_weighted(y, received.handle.token_slots, weights)

A row in 8 bits is a record: its e4m3 values, then one fp32 scale for every 128 columns, padded to a multiple of
512 bytes.  A value stands for itself times its group's scale, and a scale is the largest magnitude of its group over 448.
The buffer that dispatches records is one whose `hidden` is `fp8_payload_width(hidden)`.

Calls run on the caller's current stream; nothing is copied to the host.  `ValueError` for misuse of arguments, as
`Buffer` has it; `RuntimeError` where a derivative is asked for that an operator does not have; in forward mode none has one.
None of this has a counterpart in the reference, whose experts are the caller's.
"""

from __future__ import annotations

import dataclasses
from typing import Optional

import torch

from ._native import load_extension

__all__ = [
    "Fp8Rows",
    "Fp8Weight",
    "RmsNormResult",
    "combine_weighted",
    "combine_weighted_backward",
    "dispatch_rows",
    "experts_gated",
    "experts_linear",
    "fp8_payload_width",
    "quantize_weight",
    "rms_norm_fp8",
]

SCALE_BLOCK = 128
LARGEST_FP8 = 448.0
SMALLEST_AMAX = 2.0**-64  # a group whose values are all smaller has the scale of this one
RECORD_ALIGNMENT = 512


def _record_bytes(columns: int) -> int:
    used = columns + 4 * (-(-columns // SCALE_BLOCK))
    return -(-used // RECORD_ALIGNMENT) * RECORD_ALIGNMENT


def fp8_payload_width(hidden: int) -> int:
    """bf16 elements that a record of `hidden` values takes: the `hidden` of the buffer that dispatches it."""
    if isinstance(hidden, bool) or not isinstance(hidden, int) or hidden <= 0 or hidden % 16:
        raise ValueError("hidden must be a positive multiple of 16")
    return _record_bytes(hidden) // 2


@dataclasses.dataclass
class Fp8Rows:
    """Rows in 8 bits.

    values    float8_e4m3fn [rows, hidden], rows a multiple of 16 bytes apart
    scales    float32 [rows, ceil(hidden / 128)]
    payload   bf16 [rows, fp8_payload_width(hidden)]: the records that the two are views of, None when they are
              tensors of their own
    """

    values: torch.Tensor
    scales: torch.Tensor
    payload: Optional[torch.Tensor] = None

    @classmethod
    def of_payload(cls, payload: torch.Tensor, hidden: int) -> "Fp8Rows":
        """The rows that a tensor of records holds (what a dispatch of `payload` returns)."""
        width = fp8_payload_width(hidden)
        if payload.dtype != torch.bfloat16 or payload.dim() != 2 or payload.shape[1] != width or not payload.is_contiguous():
            raise ValueError(f"payload must be contiguous bfloat16 [rows, {width}]")
        if payload.storage_offset() % 2:
            raise ValueError("payload must start at a whole fp32 of its storage, as its scales do")
        first = hidden // 4
        scales = payload.view(torch.float32)[:, first : first + -(-hidden // SCALE_BLOCK)]
        return cls(payload.view(torch.float8_e4m3fn)[:, :hidden], scales, payload)


@dataclasses.dataclass
class Fp8Weight:
    """Every expert's weight in 8 bits: values float8_e4m3fn [E, columns, inner], scales float32
    [E, ceil(columns / 128), ceil(inner / 128)], one a block of 128 x 128.  A gated weight holds its gate's columns, then
    its up projection's."""

    values: torch.Tensor
    scales: torch.Tensor


@dataclasses.dataclass
class RmsNormResult:
    """rows: the norm in 8 bits; residual: x + residual in bf16, None without one; normalized: the norm in bf16, None
    unless it was asked for."""

    rows: Fp8Rows
    residual: Optional[torch.Tensor]
    normalized: Optional[torch.Tensor]


@torch.no_grad()
def quantize_weight(weight: torch.Tensor) -> Fp8Weight:
    """A weight [E, columns, inner] of any floating type in 8 bits, as the products take it.  Meant for once, when a model is
    loaded; expert by expert, so that it needs the memory of one in fp32."""
    if weight.dim() != 3 or not weight.is_floating_point() or 0 in weight.shape:
        raise ValueError("weight must be a floating tensor [experts, columns, inner]")
    experts, columns, inner = weight.shape
    blocks, groups = -(-columns // SCALE_BLOCK), -(-inner // SCALE_BLOCK)
    values = torch.empty(weight.shape, dtype=torch.float8_e4m3fn, device=weight.device)
    scales = torch.empty(experts, blocks, groups, dtype=torch.float32, device=weight.device)
    for expert in range(experts):
        padded = torch.zeros(blocks * SCALE_BLOCK, groups * SCALE_BLOCK, dtype=torch.float32, device=weight.device)
        padded[:columns, :inner] = weight[expert]
        block = padded.view(blocks, SCALE_BLOCK, groups, SCALE_BLOCK)
        scales[expert] = block.abs().amax((1, 3)).clamp(min=SMALLEST_AMAX) / LARGEST_FP8
        block /= scales[expert][:, None, :, None]
        values[expert] = padded[:columns, :inner].to(torch.float8_e4m3fn)
    return Fp8Weight(values, scales)


def rms_norm_fp8(
    x: torch.Tensor, gamma: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6, normalized: bool = False
) -> RmsNormResult:
    """s = x + residual; n = s / sqrt(mean(s^2) + eps) * gamma, in fp32; n in 8 bits, s and (with `normalized`) n in bf16,
    each rounded once.  x and residual: contiguous bf16 [tokens, hidden], gamma: bf16 [hidden], hidden a multiple of 16 up to
    65536.  A group of 128 columns that holds an infinity or a NaN has an infinite or NaN scale."""
    payload, values, scales, total, plain = load_extension().rms_norm_fp8(x, gamma, residual, eps, normalized)
    return RmsNormResult(Fp8Rows(values, scales, payload), total, plain)


def experts_linear(
    rows: Fp8Rows, weight: Fp8Weight, expert_offsets: torch.Tensor | None = None, expert_counts: torch.Tensor | None = None
) -> torch.Tensor:
    """bf16 [rows, columns]: every row times its expert's weight, summed in fp32 and rounded once.

    Expert e has the rows [expert_offsets[e], expert_offsets[e] + expert_counts[e]), as a handle's layout says (int64 [E + 1]
    from 0 on, and [E]); rows of no expert are zero, and what they hold is not looked at.  Without the two, all rows are the only
    expert's.  inner is a multiple of 16, columns one of 8, both at most 2^24."""
    return load_extension().experts_linear(rows.values, rows.scales, weight.values, weight.scales, expert_offsets, expert_counts)


def experts_gated(
    rows: Fp8Rows, weight: Fp8Weight, expert_offsets: torch.Tensor | None = None, expert_counts: torch.Tensor | None = None
) -> Fp8Rows:
    """silu(gate) * up in 8 bits [rows, columns / 2]: `experts_linear` with a weight that holds the gate's columns, then the up
    projection's, in fp32 up to the one rounding to 8 bits.  columns / 2 is a multiple of 16."""
    payload, values, scales = load_extension().experts_gated(rows.values, rows.scales, weight.values, weight.scales, expert_offsets, expert_counts)
    return Fp8Rows(values, scales, payload)


def _dense(grad: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernels take one: contiguous, from a multiple of 16 bytes on (a part of a concatenation's is a
    contiguous view that starts anywhere)."""
    grad = grad.contiguous()
    return grad if grad.data_ptr() % 16 == 0 else grad.clone()


class _CombineWeighted(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, token_slots, weights, bias, expert_offsets, expert_counts):
        ctx.save_for_backward(y, token_slots, weights, expert_offsets, expert_counts)
        return load_extension().combine_weighted(y, token_slots, weights, bias, expert_offsets, expert_counts)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        y, token_slots, weights, expert_offsets, expert_counts = ctx.saved_tensors
        grad_y = grad_weights = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[2]:
            grad_y, grad_weights = combine_weighted_backward(_dense(grad), y, token_slots, weights, expert_offsets, expert_counts)
        return grad_y, None, grad_weights, grad if ctx.needs_input_grad[3] else None, None, None


def combine_weighted(
    y: torch.Tensor,
    token_slots: torch.Tensor,
    weights: torch.Tensor,
    *,
    bias: torch.Tensor | None = None,
    expert_offsets: torch.Tensor | None = None,
    expert_counts: torch.Tensor | None = None,
) -> torch.Tensor:
    """bf16 [tokens, hidden]: out[t] = bias[t] + sum over k of weights[t, k] * y[token_slots[t, k]], in fp32 in ascending k,
    rounded once.  `token_slots` is an expanded handle's int32 [tokens, topk]; a choice outside y's rows counts as
    masked, and neither its weight nor any row is looked at for it.

    It has a gradient in y, weights and bias.  The rows of y that no choice names have the gradient zero: all rows are cleared
    first.  With the layout's `expert_offsets` and `expert_counts` only the rows of no expert are: give the two with their
    handle's own `token_slots`, in which a choice names every expert's row, and not with a table that leaves some out."""
    tracked = y.requires_grad or weights.requires_grad or (bias is not None and bias.requires_grad)
    if tracked and torch.is_grad_enabled():
        return _CombineWeighted.apply(y, token_slots, weights, bias, expert_offsets, expert_counts)
    return load_extension().combine_weighted(y, token_slots, weights, bias, expert_offsets, expert_counts)


def combine_weighted_backward(
    grad: torch.Tensor,
    y: torch.Tensor,
    token_slots: torch.Tensor,
    weights: torch.Tensor,
    expert_offsets: torch.Tensor | None = None,
    expert_counts: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The gradients (grad_y bf16 [rows, hidden], grad_weights float32 [tokens, topk]) of `combine_weighted`:
    grad_y[token_slots[t, k]] = weights[t, k] * grad[t], grad_weights[t, k] = <y[token_slots[t, k]], grad[t]>, zero where masked.
    No two choices name the same row.  Without a gradient of its own."""
    return load_extension().combine_weighted_backward(grad, y, token_slots, weights, expert_offsets, expert_counts)


class _DispatchRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, buffer, handle):
        ctx.buffer, ctx.handle = buffer, handle
        return buffer.dispatch(x, handle=handle, zero_padding=handle.do_expand).x

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return ctx.buffer.combine(_dense(grad), ctx.handle).x, None, None


def dispatch_rows(buffer, x: torch.Tensor, handle) -> torch.Tensor:
    """x's rows in the handle's receive layout, padding rows zero, with a gradient: `dispatch` through the handle one way,
    `combine` of the rows' gradients the other."""
    return _DispatchRows.apply(x, buffer, handle)
