"""The expert layer's operators in 64 bits, row by row from their definitions, with the bounds their results are held to.

Bounds.  A sum of n products in fp32, in whatever order, is off by at most n * 2^-24 * sum |term| to first order; twice
that is allowed for how a matrix instruction rounds within.  bf16 results have to be the correct rounding of a value within
that; rounding to e4m3 adds 2^-4 of the value, or 2^-10 of its scale below the normal range.
"""

import torch

FP32 = 2.0**-24
BF16 = 2.0**-8  # half of the last of eight digits
FP8 = 2.0**-4
FP8_SMALL = 2.0**-10
BLOCK = 128
LARGEST = 448.0
SMALLEST_AMAX = 2.0**-64


def groups(columns):
    return -(-columns // BLOCK)


def group_amax(x):
    return torch.stack([x[:, g * BLOCK : (g + 1) * BLOCK].abs().amax(1) for g in range(groups(x.shape[1]))], 1)


def spread(scales, columns):
    """Scales of groups of 128 columns as one a column."""
    return scales.repeat_interleave(BLOCK, -1)[..., :columns]


def quantize_rows(x):
    """fp32 rows in 8 bits and their scales, for inputs of the tests."""
    scales = group_amax(x).clamp(min=SMALLEST_AMAX) / LARGEST
    return (x / spread(scales, x.shape[1])).to(torch.float8_e4m3fn), scales.float()


def check_eight_bits(values, scales, want, slack):
    """8-bit results against the exact values before their rounding, themselves known to within `slack`."""
    columns = want.shape[1]
    want_scales = group_amax(want).clamp(min=SMALLEST_AMAX) / LARGEST
    scale_slack = group_amax(slack) / LARGEST + 4 * FP32 * want_scales
    assert scales.shape == want_scales.shape and scales.dtype == torch.float32
    assert ((scales.double() - want_scales).abs() <= scale_slack).all()
    scale = spread(scales.double(), columns)
    got = values.double() * scale
    bound = torch.maximum((want.abs() + slack) * FP8, scale * FP8_SMALL) * (1 + 8 * FP32) + slack
    assert ((got - want).abs() <= bound).all()


def rms_norm(x, residual, gamma, eps):
    """s, n and a bound of n's error in fp32."""
    s = x.double() + (0 if residual is None else residual.double())
    n = s / torch.sqrt((s * s).mean(1, keepdim=True) + eps) * gamma.double()
    # the sum of squares is off by at most hidden * 2^-24 of itself, its root by half of that; a few more roundings
    return s, n, n.abs() * FP32 * (x.shape[1] / 2 + 8)


def experts(values, scales, weight, weight_scales, offsets, counts):
    """z and a bound of its error in fp32; rows of no expert are zero."""
    rows, inner = values.shape
    columns = weight.shape[1]
    z = torch.zeros(rows, columns, dtype=torch.float64)
    slack = torch.zeros_like(z)
    for e in range(weight.shape[0]):
        begin, count = (0, rows) if offsets is None else (int(offsets[e]), int(counts[e]))
        if count == 0:
            continue
        part = slice(begin, begin + count)
        a = values[part].double() * spread(scales[part].double(), inner)
        w = weight[e].double() * spread(weight_scales[e].double().repeat_interleave(BLOCK, 0)[:columns], inner)
        z[part] = a @ w.T
        slack[part] = 2 * (inner + groups(inner)) * FP32 * (a.abs() @ w.abs().T)
    return z, slack


def gated(z, slack):
    """silu(gate) * up and a bound of its error: |silu'| <= 1.1, a few roundings, and 2^-21 of the exponential."""
    half = z.shape[1] // 2
    gate, up = z[:, :half], z[:, half:]
    act = gate * torch.sigmoid(gate) * up
    # (the exponential's argument is rounded: a relative error of |gate| * 2^-24 in it)
    off = 1.1 * slack[:, :half] * up.abs() + gate.abs() * slack[:, half:] + act.abs() * (2.0**-21 + FP32 * gate.abs())
    return act, off


def combine(y, slots, weights, bias):
    tokens, topk = slots.shape
    out = torch.zeros(tokens, y.shape[1], dtype=torch.float64)
    slack = torch.zeros_like(out)
    for t in range(tokens):
        for k in range(topk):
            slot = int(slots[t, k])
            if 0 <= slot < y.shape[0]:
                term = weights[t, k].double() * y[slot].double()
                out[t] += term
                slack[t] += term.abs()
        if bias is not None:
            out[t] += bias[t].double()
            slack[t] += bias[t].double().abs()
    return out, slack * FP32 * (topk + 1)


def combine_backward(grad, y, slots, weights):
    tokens, topk = slots.shape
    grad_y = torch.zeros(y.shape, dtype=torch.float64)
    grad_weights = torch.zeros(weights.shape, dtype=torch.float64)
    slack = torch.zeros_like(grad_weights)
    for t in range(tokens):
        for k in range(topk):
            slot = int(slots[t, k])
            if 0 <= slot < y.shape[0]:
                grad_y[slot] = weights[t, k].double() * grad[t].double()
                terms = y[slot].double() * grad[t].double()
                grad_weights[t, k] = terms.sum()
                slack[t, k] = terms.abs().sum() * FP32 * y.shape[1]
    return grad_y, grad_weights, slack
