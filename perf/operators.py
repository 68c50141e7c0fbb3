"""The expert layer's operators around dispatch and combine, as cases that can be timed.

A case is one call of one operator, by its `op`:

  norm              residual addition and root-mean-square norm of a batch's rows, in 8 bits with a scale for
                    every 128 columns (the layer's entry; the rows then go through dispatch)
  gated             the experts' first product: dispatched 8-bit rows times every expert's gate and up
                    projections (8 bits, one scale a 128 x 128 block), silu(gate) * up, in 8 bits again
  linear            the experts' second product: the same rows times every expert's down projection, bf16
  combine           every token's expert rows brought back, multiplied by their gate weights and summed
  combine_backward  its gradient: of the expert rows and of the gate weights

Rows are in expert-major segments, as dispatch leaves them.  Row tensors in 8 bits are what dispatch moves:
one record a row, its values, then its scales.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 128               # columns that share a scale; weights: 128 x 128
LARGEST = 448.0           # largest finite e4m3 value
SMALLEST_AMAX = 2.0**-64  # a group whose values are all smaller has the scale of this one
EPS = 1e-6
MASKED_SHARE = 0.1

# Routing kinds, as in the repository's workloads:
#   uniform   K distinct experts, all equally likely
#   dropout   top-K of normal logits, a tenth of the choices masked (-1)
#   biased    top-K of normal logits plus a per-expert bias of deviation 2
ROUTINGS = ("uniform", "dropout", "biased")


def _norm(name, tokens, hidden, *, residual=True, normalized=True):
    return {"name": name, "op": "norm", "tokens": tokens, "hidden": hidden, "residual": residual, "normalized": normalized}


def _product(name, op, tokens, topk, experts, inner, columns, *, routing="dropout", alignment=1):
    return {"name": name, "op": op, "tokens": tokens, "topk": topk, "experts": experts, "inner": inner, "columns": columns,
            "routing": routing, "alignment": alignment}


def _weighted(name, op, tokens, hidden, experts, topk, *, routing="dropout", alignment=1, bias=False):
    return {"name": name, "op": op, "tokens": tokens, "hidden": hidden, "experts": experts, "topk": topk, "routing": routing,
            "alignment": alignment, "bias": bias}


def listed():
    return [
        # one sequence's next token: the smallest call, all latency
        _norm("norm-token", 1, 7168, normalized=False),
        # a prefill batch of 4096 x 7168, whose router reads the norm's output too
        _norm("norm-prefill", 4096, 7168),
        # one token's eight experts of 64: every weight row is read for one activation row
        _product("gated-token", "gated", 1, 8, 64, 7168, 4096, routing="uniform"),
        # a decode step with 256 tokens in flight: some 29 rows an expert
        _product("gated-decode", "gated", 256, 8, 64, 4096, 4096),
        # one rank's 32 experts in a prefill: some 900 rows an expert, the largest product
        _product("gated-prefill", "gated", 4096, 8, 32, 7168, 4096, alignment=128),
        # a decode step of narrow experts, most of them with one or two rows
        _product("linear-decode", "linear", 16, 8, 128, 768, 2048),
        # odd sizes: columns that end inside a block, uneven segments that start anywhere
        _product("linear-ragged", "linear", 1537, 6, 60, 1424, 2816, routing="biased", alignment=16),
        # the second product of the prefill
        _product("linear-prefill", "linear", 4096, 8, 32, 2048, 7168, alignment=128),
        # the decode step's rows brought back
        _weighted("combine-decode", "combine", 256, 4096, 64, 8),
        # a prefill batch's rows brought back, a shared expert's output added
        _weighted("combine-prefill", "combine", 4096, 7168, 256, 8, bias=True),
        # gradients of an odd batch with padded segments
        _weighted("backward-ragged", "combine_backward", 1537, 2816, 60, 6, routing="biased", alignment=16),
        # gradients of a training batch, segments padded for the products
        _weighted("backward-batch", "combine_backward", 4096, 7168, 256, 8, alignment=128),
    ]


def draw(rng):
    """A case of the ranges above: 1 to 8192 tokens, rows of 256 to 7168 values, 1 to 256 experts of 128 to 8192
    columns, one to eight choices a token."""
    most = {"bytes": 0, "flops": 0}
    for case in listed():
        for key, value in work(case).items():
            most[key] = max(most[key], value)

    def spread(low, high, step=1):
        return step * int(round(math.exp(rng.uniform(math.log(low / step), math.log(high / step)))))

    while True:
        op = rng.choice(("norm", "gated", "linear", "combine", "combine_backward"))
        tokens = spread(1, 8192)
        if op == "norm":
            case = _norm("", tokens, spread(256, 7168, 16), residual=rng.random() < 0.7, normalized=rng.random() < 0.5)
            sizes = (tokens, case["hidden"])
        else:
            experts = spread(1, 256)
            topk = rng.choice([k for k in (1, 2, 3, 4, 6, 8) if k <= experts])
            # (a batch of a few choices that were all masked would have no outputs)
            routing = rng.choice(ROUTINGS if tokens * topk >= 16 else ("uniform", "biased"))
            alignment = rng.choice((1, 1, 16, 128))
            if op in ("gated", "linear"):
                inner, columns = spread(256, 7168, 16), spread(128, 4096, 16)
                columns *= 2 if op == "gated" else 1
                case = _product("", op, tokens, topk, experts, inner, columns, routing=routing, alignment=alignment)
                if experts * inner * columns > 64 * 7168 * 4096:
                    continue
                sizes = (tokens, inner, columns, columns // 2)
            else:
                case = _weighted("", op, tokens, spread(256, 7168, 8), experts, topk, routing=routing, alignment=alignment,
                                 bias=op == "combine" and rng.random() < 0.4)
                sizes = (tokens, case["hidden"])
        del case["name"]
        if 3072 not in sizes and all(value <= most[key] for key, value in work(case).items()):
            return case


# ------------------------------------------------------------------ inputs


def _routing(case, generator):
    """Expert ids [T, K], -1 where masked, and gate weights [T, K]."""
    # The batch's load (how many choices each expert gets, how many are masked) belongs to the case, so that
    # the outputs have the case's shapes; the seed decides which token and which expert is which.
    tokens, experts, topk = case["tokens"], case["experts"], case["topk"]
    load = torch.Generator(device="cuda").manual_seed(20)
    logits = torch.randn(tokens, experts, device="cuda", generator=load)
    if case["routing"] == "biased":
        logits = logits + 2.0 * torch.randn(experts, device="cuda", generator=load)
    token_of = torch.randperm(tokens, device="cuda", generator=generator)
    expert_of = torch.randperm(experts, device="cuda", generator=generator)
    chosen, ids = logits.topk(topk, dim=1)
    ids, weights = expert_of[ids][token_of], torch.softmax(chosen, dim=1)[token_of]
    if case["routing"] == "dropout":
        masked = torch.rand(tokens, topk, device="cuda", generator=load) < MASKED_SHARE
        ids = ids.masked_fill(masked[token_of], -1)
    return ids, weights.contiguous()


def _layout(ids, experts, alignment):
    """Slots [T, K] (int32, -1 where masked), counts [E] and offsets [E + 1] (int64) of the expert-major rows, and their number."""
    flat = ids.reshape(-1)
    counts = torch.bincount(flat[flat >= 0], minlength=experts)
    padded = (counts + alignment - 1) // alignment * alignment
    offsets = torch.cat([torch.zeros_like(padded[:1]), padded.cumsum(0)])
    before = counts.cumsum(0) - counts
    key = torch.where(flat >= 0, flat, experts)
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(flat.numel(), device="cuda")
    named = flat.clamp(min=0)
    slots = torch.where(flat >= 0, offsets[named] + place - before[named], -1)
    return slots.to(torch.int32).reshape(ids.shape), counts, offsets, int(offsets[-1])


def _records(rows, columns):
    """Empty row records: their bytes, and the views of them that hold values and scales."""
    groups = -(-columns // BLOCK)
    size = -(-(columns + 4 * groups) // 512) * 512
    record = torch.zeros(rows, size, dtype=torch.uint8, device="cuda")
    return record[:, :columns].view(torch.float8_e4m3fn), record.view(torch.float32)[:, columns // 4 : columns // 4 + groups]


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=generator)

    op, state = case["op"], {"case": dict(case)}
    if op == "norm":
        shape = (case["tokens"], case["hidden"])
        # a few channels are much larger than the rest, as in a trained model's residual stream
        loud = 1.0 + 20.0 * (torch.rand(case["hidden"], device="cuda", generator=generator) < 0.01)
        state["x"] = (normal(*shape) * loud).to(torch.bfloat16)
        state["residual"] = (2.0 * normal(*shape) * loud).to(torch.bfloat16) if case["residual"] else None
        state["gamma"] = (1.0 + 0.1 * normal(case["hidden"])).to(torch.bfloat16)
        return state
    ids, weights = _routing(case, generator)
    slots, counts, offsets, rows = _layout(ids, case["experts"], case["alignment"])
    state.update(counts=counts, offsets=offsets)
    if op in ("gated", "linear"):
        inner, columns, experts = case["inner"], case["columns"], case["experts"]
        groups, blocks = -(-inner // BLOCK), -(-columns // BLOCK)
        state["values"], state["scales"] = _records(rows, inner)
        live = slots[slots >= 0].long()
        x = torch.zeros(live.numel(), groups * BLOCK, device="cuda")
        x[:, :inner] = normal(live.numel(), inner)
        x = x.view(-1, groups, BLOCK)
        scales = x.abs().amax(2).clamp(min=SMALLEST_AMAX) / LARGEST
        values = (x / scales[:, :, None]).to(torch.float8_e4m3fn).view(-1, groups * BLOCK)[:, :inner]
        state["values"].view(torch.uint8)[live] = values.view(torch.uint8)
        state["scales"][live] = scales
        weight = torch.empty(experts, columns, inner, dtype=torch.float8_e4m3fn, device="cuda")
        weight_scales = torch.empty(experts, blocks, groups, device="cuda")
        for expert in range(experts):
            w = torch.zeros(blocks * BLOCK, groups * BLOCK, device="cuda")
            w[:columns, :inner] = normal(columns, inner) / math.sqrt(inner)
            w = w.view(blocks, BLOCK, groups, BLOCK)
            weight_scales[expert] = w.abs().amax((1, 3)).clamp(min=SMALLEST_AMAX) / LARGEST
            w = (w / weight_scales[expert][:, None, :, None]).to(torch.float8_e4m3fn).view(blocks * BLOCK, groups * BLOCK)
            weight.view(torch.uint8)[expert] = w[:columns, :inner].view(torch.uint8)
        state.update(weight=weight, weight_scales=weight_scales)
        return state
    state.update(slots=slots, weights=weights, y=normal(rows, case["hidden"]).to(torch.bfloat16))
    if op == "combine":
        state["bias"] = normal(case["tokens"], case["hidden"]).to(torch.bfloat16) if case["bias"] else None
    else:
        state["grad"] = normal(case["tokens"], case["hidden"]).to(torch.bfloat16)
    return state


# ------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(op, state)
    if op == "norm":
        return _plain_norm(**state)
    if op == "combine":
        return _plain_combine(**state)
    if op == "combine_backward":
        return _plain_combine_backward(**state)
    y = _plain_product(**state)
    if op == "linear":
        return {"y": y.to(torch.bfloat16)}
    gate, up = y.chunk(2, dim=1)
    values, scales = _quantized(gate / (1.0 + torch.exp(-gate)) * up)
    return {"values": values, "scales": scales}


def _run_own(op, state):
    import nanoep_amd as ep

    if op == "norm":
        result = ep.rms_norm_fp8(state["x"], state["gamma"], residual=state["residual"], eps=EPS, normalized=state["case"]["normalized"])
        return {"values": result.rows.values, "scales": result.rows.scales, "residual": result.residual, "normalized": result.normalized}
    if op == "combine":
        return {"out": ep.combine_weighted(state["y"], state["slots"], state["weights"], bias=state["bias"])}
    if op == "combine_backward":
        grad_y, grad_weights = ep.combine_weighted_backward(state["grad"], state["y"], state["slots"], state["weights"],
                                                            state["offsets"], state["counts"])
        return {"grad_y": grad_y, "grad_weights": grad_weights}
    rows, weight = ep.Fp8Rows(state["values"], state["scales"]), ep.Fp8Weight(state["weight"], state["weight_scales"])
    if op == "linear":
        return {"y": ep.experts_linear(rows, weight, state["offsets"], state["counts"])}
    out = ep.experts_gated(rows, weight, state["offsets"], state["counts"])
    return {"values": out.values, "scales": out.scales}


def _quantized(x):
    """x in 8 bits and the scales of its groups of 128 columns."""
    columns = x.shape[1]
    x = torch.nn.functional.pad(x, (0, -columns % BLOCK)).view(x.shape[0], -1, BLOCK)
    scales = x.abs().amax(2).clamp(min=SMALLEST_AMAX) / LARGEST
    return (x / scales[:, :, None]).view(x.shape[0], -1)[:, :columns].to(torch.float8_e4m3fn), scales


def _plain_norm(case, x, residual, gamma):
    s = x.float() if residual is None else x.float() + residual.float()
    n = s * torch.rsqrt(s.square().mean(dim=1, keepdim=True) + EPS) * gamma.float()
    values, scales = _quantized(n)
    return {"values": values, "scales": scales, "residual": None if residual is None else s.to(torch.bfloat16),
            "normalized": n.to(torch.bfloat16) if case["normalized"] else None}


def _plain_product(case, values, scales, weight, weight_scales, counts, offsets):
    """y [rows, columns] in 32 bits, zero in rows of no expert: the experts that have rows, padded to the longest, as one batched product."""
    rows, columns, inner = values.shape[0], weight.shape[1], weight.shape[2]
    active = counts.nonzero()[:, 0]
    slot = torch.arange(rows, device="cuda")
    expert = torch.searchsorted(offsets[1:], slot, right=True)
    place = slot - offsets[expert]
    live = (place < counts[expert]).nonzero()[:, 0]
    index = torch.zeros_like(counts)
    index[active] = torch.arange(active.numel(), device="cuda")
    batch, place = index[expert[live]], place[live]
    padded = torch.zeros(active.numel(), int(counts.max()), inner, device="cuda")
    padded[batch, place] = values[live].float() * scales[live].repeat_interleave(BLOCK, 1)[:, :inner]
    w = weight[active].float()
    w *= weight_scales[active].repeat_interleave(BLOCK, 1)[:, :columns].repeat_interleave(BLOCK, 2)[:, :, :inner]
    y = torch.zeros(rows, columns, device="cuda")
    y[live] = torch.bmm(padded, w.transpose(1, 2))[batch, place]
    return y


def _plain_combine(case, y, slots, weights, bias, counts, offsets):
    chosen = y[slots.clamp(min=0)].float()
    out = (chosen * torch.where(slots >= 0, weights, 0.0)[:, :, None]).sum(1)
    return {"out": (out if bias is None else out + bias.float()).to(torch.bfloat16)}


def _plain_combine_backward(case, y, slots, weights, grad, counts, offsets):
    token, choice = (slots >= 0).nonzero(as_tuple=True)
    slot, g = slots[token, choice].long(), grad[token].float()
    grad_y = torch.zeros(y.shape, device="cuda", dtype=torch.bfloat16)
    grad_y[slot] = (g * weights[token, choice][:, None]).to(torch.bfloat16)
    grad_weights = torch.zeros_like(weights)
    grad_weights[token, choice] = (y[slot].float() * g).sum(1)
    return {"grad_y": grad_y, "grad_weights": grad_weights}


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]

    def eight_bits(x):
        # values before their rounding to 8 bits
        columns = x.shape[1]
        groups = -(-columns // BLOCK)
        values, scales = torch.empty_like(x), x.new_empty(x.shape[0], groups)
        for g in range(groups):
            part = x[:, g * BLOCK : (g + 1) * BLOCK]
            scales[:, g] = part.abs().max(dim=1).values.clamp(min=SMALLEST_AMAX) / LARGEST
            values[:, g * BLOCK : (g + 1) * BLOCK] = part / scales[:, g : g + 1]
        return values, scales

    if op == "norm":
        s = state["x"].double()
        if state["residual"] is not None:
            s = s + state["residual"].double()
        mean = (s * s).sum(1, keepdim=True) / s.shape[1]
        n = s / torch.sqrt(mean + EPS) * state["gamma"].double()
        values, scales = eight_bits(n)
        return {"values": values, "scales": scales, "residual": None if state["residual"] is None else s,
                "normalized": n if case["normalized"] else None}
    if op == "combine":
        total = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
        for k in range(case["topk"]):
            token = (state["slots"][:, k] >= 0).nonzero()[:, 0]
            total[token] += state["weights"][token, k].double()[:, None] * state["y"][state["slots"][token, k].long()].double()
        if state["bias"] is not None:
            total += state["bias"].double()
        return {"out": total}
    if op == "combine_backward":
        grad_y = torch.zeros(state["y"].shape, dtype=torch.float64, device="cuda")
        grad_weights = torch.zeros(state["weights"].shape, dtype=torch.float64, device="cuda")
        for k in range(case["topk"]):
            token = (state["slots"][:, k] >= 0).nonzero()[:, 0]
            slot = state["slots"][token, k].long()
            grad_y[slot] = state["weights"][token, k].double()[:, None] * state["grad"][token].double()
            grad_weights[token, k] = (state["y"][slot].double() * state["grad"][token].double()).sum(1)
        return {"grad_y": grad_y, "grad_weights": grad_weights}
    rows, inner, columns = state["values"].shape[0], case["inner"], case["columns"]
    y = torch.zeros(rows, columns, dtype=torch.float64, device="cuda")
    starts, counts = state["offsets"].tolist(), state["counts"].tolist()
    row_scale = torch.arange(inner, device="cuda") // BLOCK
    column_scale = torch.arange(columns, device="cuda") // BLOCK
    for expert, count in enumerate(counts):
        if count:
            part = slice(starts[expert], starts[expert] + count)
            a = state["values"][part].double() * state["scales"][part].double()[:, row_scale]
            w = state["weight"][expert].double() * state["weight_scales"][expert].double()[column_scale][:, row_scale]
            y[part] = a @ w.T
    if op == "linear":
        return {"y": y}
    gate, up = y[:, : columns // 2], y[:, columns // 2 :]
    values, scales = eight_bits(gate * torch.sigmoid(gate) * up)
    return {"values": values, "scales": scales}


# ------------------------------------------------------------------ what a pass cannot do without


def _routed_rows(case):
    """Valid choices, as an expected value of the routing, and the experts that have any."""
    assigned = case["tokens"] * case["topk"] * (1.0 - MASKED_SHARE if case["routing"] == "dropout" else 1.0)
    active = case["experts"] * (1.0 - (1.0 - 1.0 / case["experts"]) ** assigned) if case["experts"] > 1 else 1.0
    return assigned, active, assigned + min(case["experts"], assigned) * (case["alignment"] - 1) / 2.0


def work(case):
    op = case["op"]
    if op == "norm":
        values = case["tokens"] * case["hidden"]
        each = 2 + 1 + 4 / BLOCK + (4 if case["residual"] else 0) + (2 if case["normalized"] else 0)
        return {"bytes": values * each + 2 * case["hidden"], "flops": 8 * values}
    assigned, active, rows = _routed_rows(case)
    if op in ("gated", "linear"):
        inner, columns = case["inner"], case["columns"]
        read = assigned * inner * (1 + 4 / BLOCK) + active * columns * inner * (1 + 4 / BLOCK**2)
        written = rows * (columns / 2 * (1 + 4 / BLOCK) if op == "gated" else 2 * columns)
        return {"bytes": read + written, "flops": 2 * assigned * columns * inner}
    row, choices = 2 * case["hidden"], case["tokens"] * case["topk"]
    if op == "combine":
        return {"bytes": row * (assigned + case["tokens"] * (2 if case["bias"] else 1)) + 8 * choices, "flops": 2 * assigned * case["hidden"]}
    return {"bytes": row * (assigned + case["tokens"] + rows) + 12 * choices, "flops": 3 * assigned * case["hidden"]}
