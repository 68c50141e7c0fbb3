"""The operators at an expert layer's entry (norms, router, balance loss) in 64 bits on the CPU, from their definitions, with the bounds
their results are held to.

Bounds.  A sum in fp32 in which no term goes through more than D additions is off by at most D * 2^-24 * sum |term|, to first order.  The
sums within a row or a token here are trees: at most 16 additions in a lane (64 experts in one), 6 in a wavefront, 16 over a workgroup's
wavefronts, so that D = 96 covers them with the roundings of their terms.  An exponential is good to 2^-22 of itself, and its argument, a
difference, is rounded: |argument| * 2^-24 more.
"""

import math

import torch

FP32 = 2.0**-24
DEPTH = 96
EXP = 2.0**-22
LEAST = 2.0**-126  # below it fp32 loses digits


def rounding(dtype):
    return 2.0**-8 if dtype == torch.bfloat16 else FP32


def check_rounded(got, want, slack, dtype):
    """The correct rounding of some value within `slack` of the exact one."""
    assert got.shape == want.shape and got.dtype == dtype
    got = got.cpu().double()
    if dtype == torch.bfloat16:
        low, high = (want - slack).to(dtype).double(), (want + slack).to(dtype).double()
    else:
        low, high = want - slack - want.abs() * FP32 - LEAST, want + slack + want.abs() * FP32 + LEAST
    wrong = ~((low <= got) & (got <= high))
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()} values: {got[wrong][:4]} for {want[wrong][:4]}, {slack.expand_as(want)[wrong][:4]}"


# ------------------------------------------------------------------ norms


def total_of(x, residual):
    """What is normed: the sum in fp32, rounded to the rows' type."""
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def norm(s, gamma, beta, eps, centred):
    """(y, its slack), (mean, its slack), (rstd, its slack) for rows s."""
    s, gamma = s.double(), gamma.double()
    mean = s.mean(1, keepdim=True) if centred else torch.zeros_like(s[:, :1])
    mean_slack = (DEPTH + 1) * FP32 * s.abs().mean(1, keepdim=True) if centred else torch.zeros_like(mean)
    c = s - mean
    c_slack = mean_slack + FP32 * c.abs()
    var = (c * c).mean(1, keepdim=True)
    var_slack = (2 * c.abs() * c_slack + c_slack * c_slack).mean(1, keepdim=True) + (DEPTH + 2) * FP32 * var
    rstd = (var + eps).rsqrt()
    # (monotone: between its values at the ends; the square root, the quotient and the addition of eps are rounded)
    worst = torch.maximum((var - var_slack + eps).clamp(min=1e-300).rsqrt() - rstd, rstd - (var + var_slack + eps).rsqrt())
    rstd_slack = worst + 4 * FP32 * rstd
    z = c * rstd
    y = z * gamma + (0 if beta is None else beta.double())
    y_slack = (c_slack * (rstd + rstd_slack) + c.abs() * rstd_slack) * gamma.abs() + 3 * FP32 * ((z * gamma).abs() + y.abs())
    return (y, y_slack), (mean[:, 0], mean_slack[:, 0]), (rstd[:, 0], rstd_slack[:, 0])


def norm_backward(grad, total, gamma, mean, rstd, grad_residual):
    """(grad_x, its slack), (grad_gamma, its slack), (grad_beta, its slack) from fp32 statistics that are taken as they are."""
    g, gamma, rstd = grad.double(), gamma.double(), rstd.double()[:, None]
    tokens = g.shape[0]
    z = (total.double() - (0 if mean is None else mean.double()[:, None])) * rstd
    u = g * gamma
    along, along_slack = (u * z).mean(1, keepdim=True), (DEPTH + 5) * FP32 * (u * z).abs().mean(1, keepdim=True)
    across, across_slack = torch.zeros_like(along), torch.zeros_like(along)
    if mean is not None:
        across, across_slack = u.mean(1, keepdim=True), (DEPTH + 2) * FP32 * u.abs().mean(1, keepdim=True)
    x = rstd * (u - across - z * along)
    slack = rstd * (across_slack + z.abs() * along_slack + 6 * FP32 * (u.abs() + across.abs() + (z * along).abs()))
    if grad_residual is not None:
        x = x + grad_residual.double()
        slack = slack + FP32 * x.abs()
    # a term: the rows of one of at least 256 workgroups' teams, the teams, a sixteenth of the workgroups' sums, sixteen of those
    depth = min(tokens, tokens / 256 + 160) + 3
    return (x, slack), ((g * z).sum(0), depth * FP32 * (g * z).abs().sum(0)), (g.sum(0), depth * FP32 * g.abs().sum(0))


# ------------------------------------------------------------------ router


def scores(logits, scoring):
    """Every expert's score in 64 bits."""
    logits = logits.double()
    return torch.sigmoid(logits) if scoring == "sigmoid" else torch.softmax(logits, dim=1)


def choose(logits, topk, scoring, bias=None, mask=None, groups=1, topk_groups=1):
    """ids [T, K], -1 where nothing is left."""
    logits = logits.double()
    value = logits
    grouped = topk_groups < groups
    if bias is not None or grouped:
        value = scores(logits, scoring) + (0 if bias is None else bias.double())
    never = (logits == -math.inf) | (value == -math.inf)
    value = value.masked_fill(never, -math.inf)
    if grouped:
        parts = value.reshape(value.shape[0], groups, -1)
        best = parts.sort(dim=2, descending=True).values
        of_group = best[:, :, 0].clone()
        if parts.shape[2] > 1:
            of_group = torch.where(best[:, :, 1] == -math.inf, of_group, of_group + best[:, :, 1])
        kept = of_group.sort(dim=1, descending=True, stable=True).indices[:, :topk_groups]
        closed = torch.ones_like(of_group, dtype=torch.bool).scatter(1, kept, False)
        value = parts.masked_fill(closed[:, :, None], -math.inf).reshape(value.shape)
    order = value.sort(dim=1, descending=True, stable=True)
    ids = order.indices[:, :topk].masked_fill(order.values[:, :topk] == -math.inf, -1)
    return ids if mask is None else ids.masked_fill(~mask[:, None], -1)


def _spread(logits):
    """How far the finite logits of a token are from its largest, which its exponentials' arguments are rounded by."""
    finite = torch.where(logits.isfinite(), logits.double(), 0.0)
    return finite.abs().amax(1, keepdim=True) + (finite.amax(1, keepdim=True) - finite.amin(1, keepdim=True))


def weigh(logits, ids, scoring, normalize, scale):
    """weights [T, K] of given choices, and their slack."""
    logits = logits.double()
    kept, named = (ids >= 0) & (ids < logits.shape[1]), ids.clamp(0, logits.shape[1] - 1)
    chosen = torch.where(kept, logits.gather(1, named), -math.inf)
    if scoring == "sigmoid":
        s = torch.sigmoid(chosen)
        if normalize:  # by hand, because sigmoids may all be tiny
            top = chosen.amax(1, keepdim=True).clamp(max=0.0)
            top = torch.where(top == -math.inf, 0.0, top)
            s = torch.exp(chosen.clamp(max=0.0) - top) / (1 + torch.exp(-chosen.abs()))
    elif normalize:
        top = chosen.amax(1, keepdim=True)
        s = torch.exp(chosen - torch.where(top == -math.inf, 0.0, top))
    else:
        s = torch.softmax(logits, dim=1).gather(1, named)
    s = torch.where(kept, s, 0.0)
    if normalize:
        s = s / torch.where(s.sum(1, keepdim=True) > 0, s.sum(1, keepdim=True), 1.0)
    relative = 2 * (_spread(logits) * FP32 + EXP) + (DEPTH + 8) * FP32
    return s * scale, s * scale * relative + LEAST


def weigh_backward(grad, logits, ids, scoring, normalize, scale):
    """grad_logits [T, E] and its slack: every term of it to within a relative error."""
    logits, grad = logits.double(), grad.double() * scale
    experts = logits.shape[1]
    kept, named = (ids >= 0) & (ids < experts), ids.clamp(0, experts - 1)
    grad = torch.where(kept, grad, 0.0)
    relative = 3 * (_spread(logits) * FP32 + EXP) + (DEPTH + 16) * FP32
    chosen = torch.where(kept, logits.gather(1, named), 0.0)
    out, size = torch.zeros_like(logits), torch.zeros_like(logits)
    if scoring == "softmax" and not normalize:
        p = torch.softmax(logits, dim=1)
        wide = torch.zeros_like(p).scatter_add(1, named, grad)
        wide_size = torch.zeros_like(p).scatter_add(1, named, grad.abs())
        out = p * (wide - (wide * p).sum(1, keepdim=True))
        size = p * (wide_size + (wide_size * p).sum(1, keepdim=True))
        return out, size * relative + LEAST
    rest = torch.sigmoid(-chosen) if scoring == "sigmoid" else torch.ones_like(chosen)
    if normalize:
        w, _ = weigh(logits, ids, scoring, True, 1.0)
        each = w * rest * (grad - (w * grad).sum(1, keepdim=True))
        each_size = w * rest * (grad.abs() + (w * grad.abs()).sum(1, keepdim=True))
    else:
        each = grad * torch.sigmoid(chosen) * rest
        each_size = each.abs()
    each, each_size = torch.where(kept, each, 0.0), torch.where(kept, each_size, 0.0)
    out.scatter_add_(1, named, each)
    size.scatter_add_(1, named, each_size)
    return out, size * relative + LEAST


# ------------------------------------------------------------------ balance


def shares(logits, scoring):
    """Every expert's share of its token and, for sigmoids, one minus its sigmoid; zero shares for a token of -infinities."""
    logits = logits.double()
    top = logits.amax(1, keepdim=True)
    if scoring == "sigmoid":
        top = top.clamp(max=0.0)
        top = torch.where(top == -math.inf, 0.0, top)
        s, rest = torch.exp(logits.clamp(max=0.0) - top) / (1 + torch.exp(-logits.abs())), torch.sigmoid(-logits)
    else:
        s, rest = torch.exp(logits - torch.where(top == -math.inf, 0.0, top)), torch.ones_like(logits)
    total = s.sum(1, keepdim=True)
    return s / torch.where(total == 0, 1.0, total), rest


def balance(logits, ids, scoring, offsets=None, grad=None):
    """counts [S, E], tokens [S], (loss [S], its slack), and for a gradient [S] of the loss (grad_logits, its slack)."""
    rows, experts = logits.shape
    bounds = [0, rows] if offsets is None else [int(v) for v in offsets]
    count = len(bounds) - 1
    counts, tokens = torch.zeros(count, experts, dtype=torch.int64), torch.zeros(count, dtype=torch.int64)
    loss, loss_slack = torch.zeros(count, dtype=torch.float64), torch.zeros(count, dtype=torch.float64)
    found, slack = torch.zeros(rows, experts, dtype=torch.float64), torch.zeros(rows, experts, dtype=torch.float64)
    for s in range(count):
        part = slice(bounds[s], max(bounds[s], bounds[s + 1]))
        kept = (ids[part] >= 0) & (ids[part] < experts)
        live = kept.any(1)
        counts[s] = torch.bincount(ids[part][kept], minlength=experts)
        tokens[s] = live.sum()
        if not live.any():
            continue
        p, rest = shares(logits[part][live], scoring)
        relative = 2 * (_spread(logits[part][live]) * FP32 + EXP) + (DEPTH + 8) * FP32
        factor = experts * counts[s].double() / counts[s].sum() / tokens[s]
        loss[s] = (factor * p.sum(0)).sum()
        # sums over tokens and experts of terms that are all positive
        loss_slack[s] = loss[s] * (relative.max() + (int(tokens[s]) / 1024 + 300) * FP32)
        if grad is not None:
            f = factor * float(grad[s])
            along = (f * p).sum(1, keepdim=True)
            where = torch.arange(part.start, part.stop)[live]
            found[where] = p * rest * (f - along)
            slack[where] = p * rest * (f.abs() + along.abs()) * (2 * relative + 16 * FP32) + LEAST
    return counts, tokens, (loss, loss_slack), (found, slack)
