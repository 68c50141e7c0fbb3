"""The entry of an expert layer (its norm, its router, the loss that balances the experts) and their gradients, as cases
that can be timed.

A case is one call of one operator, by its `op` (for balance: the call and its gradient, as a training step makes them):

  norm            residual addition, then layer norm or root-mean-square norm of a batch's rows
  norm_backward   its gradient: of the rows (with what arrives for the sum added) and of the norm's parameters
  route           every token's experts and gate weights from its router logits, as dispatch takes them
  route_backward  the gradient of the gate weights in the logits
  balance         how many choices each expert got, the loss that grows as they get uneven, and its gradient in the logits
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
MASKED_SHARE = 0.1
PADDED_SHARE = 0.125
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _norm(name, op, kind, tokens, hidden, *, rows="bf16", parameters="bf16", residual=True):
    return {"name": name, "op": op, "kind": kind, "tokens": tokens, "hidden": hidden, "rows": rows, "parameters": parameters,
            "residual": residual}


def _route(name, op, tokens, experts, topk, *, scoring="softmax", logits="fp32", normalize=True, bias=False, groups=1, topk_groups=1,
           padded=False):
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "topk": topk, "scoring": scoring, "logits": logits,
            "normalize": normalize, "bias": bias, "groups": groups, "topk_groups": topk_groups, "padded": padded}


def _balance(name, tokens, experts, topk, *, scoring="softmax", logits="fp32", sequences=0):
    return {"name": name, "op": "balance", "tokens": tokens, "experts": experts, "topk": topk, "scoring": scoring, "logits": logits,
            "sequences": sequences}


def listed():
    return [
        # one sequence's next token: the smallest calls, all latency
        _norm("norm-token", "norm", "layer", 1, 7168),
        _route("route-token", "route", 1, 256, 8, scoring="sigmoid", bias=True, groups=8, topk_groups=4),
        # a decode step of a fixed batch size, its last tokens padding, logits as a bf16 product left them
        _route("route-decode", "route", 256, 64, 8, logits="bf16", padded=True),
        # a prefill batch of 4096 x 7168 that enters the layer
        _norm("norm-prefill", "norm", "layer", 4096, 7168),
        # ... and is routed within the best four of eight groups of experts, with a bias that evens their load
        _route("route-prefill", "route", 4096, 256, 8, scoring="sigmoid", bias=True, groups=8, topk_groups=4),
        # the longest batch, few experts, weights as the softmax over all of them left them
        _route("route-batch", "route", 32768, 64, 8, normalize=False),
        # gradients of an odd batch with a tenth of the choices masked
        _route("route-backward-ragged", "route_backward", 1537, 60, 6, logits="bf16"),
        _route("route-backward-batch", "route_backward", 8192, 128, 8, normalize=False),
        # one loss a sequence of a packed batch, sequences of uneven lengths
        _balance("balance-sequences", 8192, 128, 8, scoring="sigmoid", sequences=17),
        # one loss for the longest batch
        _balance("balance-batch", 32768, 64, 8),
        # gradients of an odd batch whose norm keeps its parameters in 32 bits
        _norm("norm-backward-ragged", "norm_backward", "rms", 1537, 2816, parameters="fp32", residual=False),
        # gradients of a training batch, the residual stream's gradient added
        _norm("norm-backward-batch", "norm_backward", "layer", 4096, 7168),
    ]


def draw(rng):
    """A case of the ranges above: 1 to 32768 tokens, rows of 256 to 7168 values, 8 to 256 experts, one to eight choices a token."""
    most = {"bytes": 0, "flops": 0}
    for case in listed():
        for key, value in work(case).items():
            most[key] = max(most[key], value)

    def spread(low, high, step=1):
        return step * int(round(math.exp(rng.uniform(math.log(low / step), math.log(high / step)))))

    while True:
        op = rng.choice(("norm", "norm_backward", "route", "route_backward", "balance"))
        # (gradients are a training batch's: not of a few tokens)
        tokens = spread(1 if op in ("norm", "route") else 64, 32768)
        if op in ("norm", "norm_backward"):
            rows, parameters = rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")))
            case = _norm("", op, rng.choice(("layer", "rms")), tokens, spread(256, 7168, 8), rows=rows, parameters=parameters,
                         residual=rng.random() < 0.6)
        else:
            experts = spread(8, 256)
            topk, scoring = rng.choice((1, 2, 3, 4, 6, 8)), rng.choice(("softmax", "sigmoid"))
            logits = rng.choice(("fp32", "fp32", "bf16"))
            if op == "balance":
                sequences = rng.choice((0, 0, spread(1, min(tokens, 64))))
                case = _balance("", tokens, experts, topk, scoring=scoring, logits=logits, sequences=sequences)
            else:
                case = _route("", op, tokens, experts, topk, scoring=scoring, logits=logits, normalize=rng.random() < 0.6)
                if op == "route":
                    case["bias"], case["padded"] = rng.random() < 0.4, tokens >= 16 and rng.random() < 0.3
                    if rng.random() < 0.4:
                        groups = rng.choice((2, 4, 8))
                        case["experts"] = max(experts // groups, 2) * groups
                        case["groups"] = groups
                        case["topk_groups"] = next(kept for kept in range(max(1, groups // 2), groups + 1)
                                                   if kept * (case["experts"] // groups) >= topk)
        del case["name"]
        if all(value <= most[key] for key, value in work(case).items()):
            return case


# ------------------------------------------------------------------ inputs


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=generator)

    op, tokens, state = case["op"], case["tokens"], {"case": dict(case)}
    if op in ("norm", "norm_backward"):
        shape, rows, parameters = (tokens, case["hidden"]), TYPES[case["rows"]], TYPES[case["parameters"]]
        layer = case["kind"] == "layer"
        # a few channels are much larger than the rest, as in a trained model's residual stream
        loud = 1.0 + 20.0 * (torch.rand(case["hidden"], device="cuda", generator=generator) < 0.01)
        x = (normal(*shape) * loud + 0.1).to(rows)
        state["gamma"] = (1.0 + 0.1 * normal(case["hidden"])).to(parameters)
        if op == "norm":
            state["x"] = x
            state["beta"] = (0.1 * normal(case["hidden"])).to(parameters) if layer else None
            state["residual"] = (2.0 * normal(*shape) * loud).to(rows) if case["residual"] else None
            return state
        state.update(total=x, grad=normal(*shape).to(rows), grad_residual=normal(*shape).to(rows) if case["residual"] else None)
        # the statistics that the norm itself left behind
        wide = x.double()
        mean = wide.mean(1) if layer else torch.zeros(tokens, dtype=torch.float64, device="cuda")
        state["rstd"] = ((wide - mean[:, None]).square().mean(1) + EPS).rsqrt().float()
        state["mean"] = mean.float() if layer else None
        return state
    experts, topk = case["experts"], case["topk"]
    # some experts are more popular than others
    logits = (1.5 * normal(tokens, experts) + 0.7 * normal(experts)).to(TYPES[case["logits"]])
    state["logits"] = logits
    if op == "route":
        # a bias that was raised and lowered in steps of a thousandth
        state["bias"] = (50.0 * normal(experts)).round() * 1e-3 if case["bias"] else None
        state["mask"] = None
        if case["padded"]:
            state["mask"] = torch.arange(tokens, device="cuda") < tokens - int(tokens * PADDED_SHARE)
        return state
    ids = logits.float().topk(topk, dim=1).indices
    masked = torch.rand(tokens, topk, device="cuda", generator=generator) < MASKED_SHARE
    state["ids"] = ids.masked_fill(masked, -1).contiguous()
    if op == "route_backward":
        state["grad"] = normal(tokens, topk)
        return state
    state["offsets"], losses = None, ()
    if case["sequences"]:
        # uneven lengths, which belong to the case; the batch's last tokens are no sequence's
        lengths = torch.rand(case["sequences"], generator=torch.Generator().manual_seed(20)).square() + 0.02
        ends = (lengths.cumsum(0) / lengths.sum() * (tokens - tokens // 50)).long()
        state["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).cuda()
        losses = (case["sequences"],)
    state["grad"] = 0.01 * (1.0 + torch.rand(losses, device="cuda", generator=generator))
    return state


# ------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(op, state)
    return {"norm": _plain_norm, "norm_backward": _plain_norm_backward, "route": _plain_route, "route_backward": _plain_route_backward,
            "balance": _plain_balance}[op](**state)


def _scale(case):
    # normalized weights of a sigmoid router add up to more than one, as its models have it
    return 2.5 if case["scoring"] == "sigmoid" else 1.0


def _run_own(op, state):
    import nanoep_amd as ep

    case = state["case"]
    if op == "norm":
        if case["kind"] == "layer":
            result = ep.layer_norm(state["x"], state["gamma"], state["beta"], residual=state["residual"], eps=EPS)
        else:
            result = ep.rms_norm(state["x"], state["gamma"], residual=state["residual"], eps=EPS)
        return {"normalized": result.normalized, "residual": result.residual, "mean": result.mean, "rstd": result.rstd}
    if op == "norm_backward":
        if case["kind"] == "layer":
            grad_x, grad_gamma, grad_beta = ep.layer_norm_backward(state["grad"], state["total"], state["gamma"], state["mean"], state["rstd"],
                                                                   grad_residual=state["grad_residual"])
            return {"grad_x": grad_x, "grad_gamma": grad_gamma, "grad_beta": grad_beta}
        grad_x, grad_gamma = ep.rms_norm_backward(state["grad"], state["total"], state["gamma"], state["rstd"],
                                                  grad_residual=state["grad_residual"])
        return {"grad_x": grad_x, "grad_gamma": grad_gamma, "grad_beta": None}
    if op == "route":
        result = ep.route_topk(state["logits"], case["topk"], scoring=case["scoring"], bias=state["bias"], mask=state["mask"],
                               groups=case["groups"], topk_groups=case["topk_groups"], normalize=case["normalize"], scale=_scale(case))
        return {"ids": result.ids, "weights": result.weights}
    if op == "route_backward":
        return {"grad_logits": ep.route_topk_backward(state["grad"], state["logits"], state["ids"], scoring=case["scoring"],
                                                      normalize=case["normalize"], scale=_scale(case))}
    result = ep.balance_loss(state["logits"], state["ids"], scoring=case["scoring"], sequence_offsets=state["offsets"])
    grad = ep.balance_loss_backward(state["grad"], state["logits"], state["ids"], result.counts, result.tokens, scoring=case["scoring"],
                                    sequence_offsets=state["offsets"])
    return {"loss": result.loss, "counts": result.counts, "tokens": result.tokens, "grad_logits": grad}


def _plain_norm(case, x, gamma, beta, residual):
    total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    s = total.float()
    mean = s.mean(dim=1, keepdim=True) if case["kind"] == "layer" else torch.zeros_like(s[:, :1])
    s = s - mean
    rstd = torch.rsqrt(s.square().mean(dim=1, keepdim=True) + EPS)
    y = s * rstd * gamma.float()
    if beta is not None:
        y = y + beta.float()
    return {"normalized": y.to(x.dtype), "residual": None if residual is None else total,
            "mean": mean[:, 0] if case["kind"] == "layer" else None, "rstd": rstd[:, 0]}


def _plain_norm_backward(case, total, gamma, grad, grad_residual, mean, rstd):
    layer = case["kind"] == "layer"
    s, g, rstd = total.float(), grad.float(), rstd[:, None]
    z = (s - mean[:, None] if layer else s) * rstd
    u = g * gamma.float()
    inner = u - z * (u * z).mean(dim=1, keepdim=True)
    if layer:
        inner = inner - u.mean(dim=1, keepdim=True)
    grad_x = inner * rstd
    if grad_residual is not None:
        grad_x = grad_x + grad_residual.float()
    return {"grad_x": grad_x.to(total.dtype), "grad_gamma": (g * z).sum(dim=0).to(gamma.dtype),
            "grad_beta": g.sum(dim=0).to(gamma.dtype) if layer else None}


def _scores(case, logits):
    """Every expert's score, in the logits' own precision."""
    if case["scoring"] == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    return e / e.sum(dim=1, keepdim=True)


def _plain_route(case, logits, bias, mask):
    logits, topk, groups = logits.float(), case["topk"], case["groups"]
    value = logits
    if bias is not None or groups > 1:
        # in 64 bits: two experts' values may be as near to one another as they like
        value = _scores(case, logits.double())
        if bias is not None:
            value = value + bias.double()
    if groups > 1:
        members = value.view(value.shape[0], groups, -1)
        best = members.sort(dim=2, descending=True).values[:, :, :2].sum(dim=2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, : case["topk_groups"]]
        dropped = torch.ones_like(best, dtype=torch.bool).scatter(1, kept, False)
        value = members.masked_fill(dropped[:, :, None], -math.inf).view_as(value)
    ids = value.sort(dim=1, descending=True, stable=True).indices[:, :topk]
    weights = _scores(case, logits).gather(1, ids)
    if case["normalize"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    weights = weights * _scale(case)
    if mask is not None:
        ids, weights = ids.masked_fill(~mask[:, None], -1), weights.masked_fill(~mask[:, None], 0.0)
    return {"ids": ids.contiguous(), "weights": weights}


def _plain_route_backward(case, logits, ids, grad):
    kept, named = ids >= 0, ids.clamp(min=0)
    scores = _scores(case, logits.float())
    chosen = scores.gather(1, named)
    # the gradient in the chosen scores
    grad = torch.where(kept, grad, 0.0) * _scale(case)
    if case["normalize"]:
        total = torch.where(kept, chosen, 0.0).sum(dim=1, keepdim=True)
        total = torch.where(total > 0, total, 1.0)
        grad = (grad - (grad * chosen).sum(dim=1, keepdim=True) / total) / total
        grad = torch.where(kept, grad, 0.0)
    wide = torch.zeros_like(scores).scatter_add(1, named, grad)
    if case["scoring"] == "sigmoid":
        return {"grad_logits": (wide * scores * (1.0 - scores)).to(logits.dtype)}
    return {"grad_logits": (scores * (wide - (wide * scores).sum(dim=1, keepdim=True))).to(logits.dtype)}


def _plain_balance(case, logits, ids, offsets, grad):
    tokens, experts = logits.shape
    if offsets is None:
        sequence, sequences = torch.zeros(tokens, dtype=torch.int64, device="cuda"), 1
    else:
        sequences = offsets.numel() - 1
        sequence = torch.searchsorted(offsets[1:], torch.arange(tokens, device="cuda"), right=True)
    kept = (ids >= 0) & (sequence < sequences)[:, None]
    live = kept.any(dim=1)
    row = sequence.clamp(max=sequences - 1)
    cells = (row[:, None] * experts + ids.clamp(min=0)).view(-1)
    counts = torch.zeros(sequences * experts, dtype=torch.int64, device="cuda").scatter_add(0, cells, kept.view(-1).long())
    counts = counts.view(sequences, experts)
    held = torch.zeros(sequences, dtype=torch.int64, device="cuda").scatter_add(0, row, live.long())
    scores = _scores(case, logits.float())
    if case["scoring"] == "sigmoid":
        shares = scores / scores.sum(dim=1, keepdim=True)
    else:
        shares = scores
    shares = shares * live[:, None]
    if offsets is None:
        mean = shares.sum(dim=0, keepdim=True)
    else:
        mean = torch.zeros(sequences, experts, device="cuda").index_add(0, row, shares)
    factor = experts * counts.float() / counts.sum(dim=1, keepdim=True).clamp(min=1) / held.clamp(min=1)[:, None]
    loss = (factor * mean).sum(dim=1)
    factor = (factor * grad.view(-1, 1))[row]
    inner = shares * (factor - (factor * shares).sum(dim=1, keepdim=True))
    if case["scoring"] == "sigmoid":
        inner = inner * (1.0 - scores)
    if offsets is None:
        loss, counts, held = loss[0], counts[0], held[0]
    return {"loss": loss, "counts": counts, "tokens": held, "grad_logits": inner.to(logits.dtype)}


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x, residual = state["x"], state["residual"]
        # the rows that are normed are those that go on, rounded as they are
        s = (x if residual is None else (x.float() + residual.float()).to(x.dtype)).double()
        mean = s.sum(1) / s.shape[1] if case["kind"] == "layer" else torch.zeros(s.shape[0], dtype=torch.float64, device="cuda")
        centred = s - mean[:, None]
        deviation = torch.sqrt((centred * centred).sum(1) / s.shape[1] + EPS)
        y = centred / deviation[:, None] * state["gamma"].double()
        if state["beta"] is not None:
            y = y + state["beta"].double()
        return {"normalized": y, "residual": None if residual is None else x.double() + residual.double(),
                "mean": mean if case["kind"] == "layer" else None, "rstd": 1.0 / deviation}
    if op == "norm_backward":
        layer = case["kind"] == "layer"
        rstd = state["rstd"].double()[:, None]
        z = state["total"].double() * rstd
        if layer:
            z = z - state["mean"].double()[:, None] * rstd
        g = state["grad"].double()
        u = g * state["gamma"].double()
        along = (u * z).sum(1, keepdim=True) / u.shape[1]
        across = u.sum(1, keepdim=True) / u.shape[1] if layer else 0.0
        grad_x = rstd * (u - across - z * along)
        if state["grad_residual"] is not None:
            grad_x = grad_x + state["grad_residual"].double()
        return {"grad_x": grad_x, "grad_gamma": (g * z).sum(0), "grad_beta": g.sum(0) if layer else None}
    logits = state["logits"].double()
    tokens, experts = logits.shape
    scores = torch.sigmoid(logits) if case["scoring"] == "sigmoid" else torch.softmax(logits, dim=1)
    if op == "route":
        value = logits.clone()
        if state["bias"] is not None:
            value = scores + state["bias"].double()
        elif case["groups"] > 1:
            value = scores.clone()
        if case["groups"] > 1:
            size = experts // case["groups"]
            of_group = torch.stack([value[:, g * size : (g + 1) * size].topk(min(2, size), dim=1).values.sum(1) for g in range(case["groups"])], 1)
            open_ = torch.zeros_like(of_group, dtype=torch.bool)
            for _ in range(case["topk_groups"]):
                best = of_group.masked_fill(open_, -math.inf).max(dim=1, keepdim=True).values
                first = ((of_group == best) & ~open_).int().argmax(dim=1, keepdim=True)
                open_.scatter_(1, first, True)
            value = value.masked_fill(~open_.repeat_interleave(size, 1), -math.inf)
        ids = torch.empty(tokens, case["topk"], dtype=torch.int64, device="cuda")
        for k in range(case["topk"]):
            best = value.max(dim=1, keepdim=True).values
            ids[:, k] = (value == best).int().argmax(dim=1)
            value.scatter_(1, ids[:, k : k + 1], -math.inf)
        weights = scores.gather(1, ids)
        if case["normalize"]:
            weights = weights / weights.sum(1, keepdim=True)
        weights = weights * _scale(case)
        if state["mask"] is not None:
            ids[~state["mask"]] = -1
            weights[~state["mask"]] = 0.0
        return {"ids": ids, "weights": weights}
    if op == "route_backward":
        # through autograd, in 64 bits
        with torch.enable_grad():
            leaf = logits.clone().requires_grad_()
            scores = torch.sigmoid(leaf) if case["scoring"] == "sigmoid" else torch.softmax(leaf, dim=1)
            kept = state["ids"] >= 0
            chosen = scores.gather(1, state["ids"].clamp(min=0)) * kept
            if case["normalize"]:
                chosen = chosen / chosen.sum(1, keepdim=True).masked_fill(~kept.any(1, keepdim=True), 1.0)
            (found,) = torch.autograd.grad(chosen, leaf, state["grad"].double() * _scale(case))
        return {"grad_logits": found}
    offsets = [0, tokens] if state["offsets"] is None else state["offsets"].tolist()
    count = len(offsets) - 1
    losses = []
    counts = torch.zeros(count, experts, dtype=torch.int64, device="cuda")
    held = torch.zeros(count, dtype=torch.int64, device="cuda")
    with torch.enable_grad():
        leaf = logits.clone().requires_grad_()
        for s in range(count):
            rows, ids = leaf[offsets[s] : offsets[s + 1]], state["ids"][offsets[s] : offsets[s + 1]]
            live = (ids >= 0).any(1)
            counts[s] = torch.bincount(ids[ids >= 0], minlength=experts)
            held[s] = live.sum()
            if case["scoring"] == "sigmoid":
                p = torch.sigmoid(rows)
                p = p / p.sum(1, keepdim=True)
            else:
                p = torch.softmax(rows, dim=1)
            mean = p[live].sum(0) / held[s].clamp(min=1)
            losses.append(experts * (counts[s].double() / counts[s].sum().clamp(min=1) * mean).sum())
        loss = torch.stack(losses)
        (found,) = torch.autograd.grad(loss, leaf, state["grad"].double().view(-1))
    loss = loss.detach()
    if state["offsets"] is None:
        loss, counts, held = loss[0], counts[0], held[0]
    return {"loss": loss, "counts": counts, "tokens": held, "grad_logits": found}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op, tokens = case["op"], case["tokens"]
    if op in ("norm", "norm_backward"):
        values, size, layer = tokens * case["hidden"], TYPES[case["rows"]].itemsize, case["kind"] == "layer"
        parameter = case["hidden"] * TYPES[case["parameters"]].itemsize * (2 if layer else 1)
        statistics = tokens * (8 if layer else 4)
        if op == "norm":
            return {"bytes": size * values * (4 if case["residual"] else 2) + parameter + statistics, "flops": 9 * values}
        return {"bytes": size * values * (4 if case["residual"] else 3) + 2 * parameter + statistics, "flops": 14 * values}
    values, choices = tokens * case["experts"], tokens * case["topk"]
    size = TYPES[case["logits"]].itemsize
    if op == "route":
        return {"bytes": size * values + 12 * choices + (4 * case["experts"] if case["bias"] else 0) + (tokens if case["padded"] else 0),
                "flops": 6 * values}
    if op == "route_backward":
        # a normalized choice's gradient needs the chosen logits only
        read = choices if case["normalize"] or case["scoring"] == "sigmoid" else values
        return {"bytes": size * (read + values) + 12 * choices, "flops": 6 * values}
    # the loss and its gradient, one after the other
    return {"bytes": size * values * 3 + 16 * choices + 16 * case["experts"] * max(1, case["sequences"]), "flops": 16 * values}
