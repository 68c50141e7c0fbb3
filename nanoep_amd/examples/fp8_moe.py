"""A mixture-of-experts layer in 8 bits, as it is served, and its gate's and rows' gradients, as it is trained, on one GPU:

    python -m nanoep_amd.examples.fp8_moe --tokens 64 --hidden 1024 --intermediate 512 --experts 16 --topk 4
    python -m nanoep_amd.examples.fp8_moe --train

Serving: the residual is added and the sum normed, in bf16 for the router and in 8 bits for the experts; the 8-bit records
go through dispatch as bf16 rows of half the length; both products read them segment by segment; the gate weights
are applied on the way back, where the shared expert's output (here: the residual) is added.  Nothing is copied to the
host between the steps.  The output is compared with a dense evaluation of the same 8-bit weights.

Training: the rows are normed and routed, go out and back through `dispatch_rows` and `combine_weighted`, and the loss that
balances the experts is added; autograd finds the gradients of all of it.  The experts in between are any differentiable function of the
rows (here: one gain a channel).
"""

from __future__ import annotations

import argparse
import json

import torch

import nanoep_amd as ep

# A product of 8-bit activations: each of them is off by at most 2^-4 of itself.
TOLERANCE = 2.0**-4
EPS = 1e-6
BALANCE = 0.01  # the balance loss's part of the objective


def make_layer(options, device):
    generator = torch.Generator().manual_seed(1)

    def normal(*shape, scale):
        return torch.randn(*shape, generator=generator) * scale

    hidden, inner = options.hidden, options.intermediate
    gate_up = normal(options.experts, 2 * inner, hidden, scale=hidden**-0.5)
    down = normal(options.experts, hidden, inner, scale=inner**-0.5)
    return {
        "gamma": (1.0 + normal(hidden, scale=0.1)).to(torch.bfloat16).to(device),
        "router": normal(options.experts, hidden, scale=hidden**-0.5).to(device),
        "gate_up": ep.quantize_weight(gate_up.to(device)),
        "down": ep.quantize_weight(down.to(device)),
    }


def route(layer, normalized, topk):
    """Expert ids [T, K] and gate weights [T, K]."""
    routing = ep.route_topk(normalized.float() @ layer["router"].T, topk)
    return routing.ids, routing.weights


def forward(buffer, layer, x, residual, options):
    """The layer's output [T, H], and what the check needs of the way there."""
    normed = ep.rms_norm_fp8(x, layer["gamma"], residual=residual, normalized=True)
    ids, weights = route(layer, normed.normalized, options.topk)
    received = buffer.dispatch(normed.rows.payload, topk_idx=ids, do_expand=True, alignment=options.alignment)
    layout = received.handle.layout
    rows = ep.Fp8Rows.of_payload(received.x, options.hidden)
    act = ep.experts_gated(rows, layer["gate_up"], layout.expert_offsets, layout.expert_counts)
    y = ep.experts_linear(act, layer["down"], layout.expert_offsets, layout.expert_counts)
    return ep.combine_weighted(y, received.handle.token_slots, weights, bias=normed.residual), normed, ids, weights


def wide(values, scales):
    """8-bit values [.., rows, columns] and their scales, a block of 128 x 128 or a group of 128 columns each, in fp32."""
    if scales.dim() == 3:
        scales = scales.repeat_interleave(128, 1)[:, : values.shape[1]]
    return values.float() * scales.repeat_interleave(128, -1)[..., : values.shape[-1]]


def dense(layer, normed, ids, weights):
    """The same, choice by choice at the source, with activations that are not rounded on the way."""
    rows = wide(normed.rows.values, normed.rows.scales)
    gate_up, down = (wide(layer[name].values, layer[name].scales) for name in ("gate_up", "down"))
    total = normed.residual.float()
    for k in range(ids.shape[1]):
        gate, up = torch.bmm(gate_up[ids[:, k]], rows[:, :, None])[:, :, 0].chunk(2, dim=1)
        act = torch.nn.functional.silu(gate) * up
        total = total + weights[:, k, None] * torch.bmm(down[ids[:, k]], act[:, :, None])[:, :, 0]
    return total


@torch.no_grad()
def serve(options):
    device = torch.device("cuda", torch.cuda.current_device())
    layer = make_layer(options, device)
    generator = torch.Generator().manual_seed(2)
    config = ep.EPConfig(options.experts, options.topk, ep.fp8_payload_width(options.hidden), max(1, options.tokens))
    with ep.Buffer(None, config) as buffer:
        for _ in range(options.steps):
            x, residual = (torch.randn(options.tokens, options.hidden, generator=generator).to(torch.bfloat16).to(device) for _ in range(2))
            got, normed, ids, weights = forward(buffer, layer, x, residual, options)
            want, base = dense(layer, normed, ids, weights), normed.residual.float()
            error = (got.float() - want).norm() / (want - base).norm()
            assert not options.tokens or error <= TOLERANCE, f"the layer is off by {float(error)}"


def train(options):
    device = torch.device("cuda", torch.cuda.current_device())
    generator = torch.Generator().manual_seed(3)
    shape = (options.tokens, options.hidden)
    x, grad = (torch.randn(*shape, generator=generator).to(torch.bfloat16).to(device) for _ in range(2))
    gains = (1.0 + 0.1 * torch.randn(options.experts, options.hidden, generator=generator)).to(torch.bfloat16).to(device)
    logits = torch.randn(options.tokens, options.experts, generator=generator).to(device)
    gamma = (1.0 + 0.1 * torch.randn(options.hidden, generator=generator)).to(device)
    leaves = [tensor.requires_grad_() for tensor in (x, gamma, gains, logits)]
    share = torch.full((), BALANCE, device=device)

    with ep.Buffer(None, ep.EPConfig(options.experts, options.topk, options.hidden, max(1, options.tokens))) as buffer:
        normed = ep.rms_norm(x, gamma, eps=EPS).normalized
        routing = ep.route_topk(logits, options.topk, normalize=False)
        handle = buffer.dispatch(normed.detach(), topk_idx=routing.ids, do_expand=True, alignment=options.alignment).handle
        layout = handle.layout
        rows = ep.dispatch_rows(buffer, normed, handle)
        slot = torch.arange(rows.shape[0], device=device)
        expert = torch.searchsorted(layout.expert_offsets[1:].contiguous(), slot, right=True).clamp(max=options.experts - 1)
        out = ep.combine_weighted(rows * gains[expert], handle.token_slots, routing.weights, expert_offsets=layout.expert_offsets,
                                  expert_counts=layout.expert_counts)
        balance = ep.balance_loss(logits, routing.ids)
        found = torch.autograd.grad((out, balance.loss), leaves, (grad, share))

    # the same in fp32, choice by choice at the source
    wide = x.float()
    wide = wide * torch.rsqrt(wide.square().mean(dim=1, keepdim=True) + EPS) * gamma
    scores = torch.softmax(logits, dim=1)
    dense_out = (wide[:, None] * gains.float()[routing.ids] * scores.gather(1, routing.ids)[:, :, None]).sum(1)
    chosen = torch.bincount(routing.ids.reshape(-1), minlength=options.experts)
    dense_balance = options.experts * (chosen / chosen.sum() * scores.mean(dim=0)).sum()
    wanted = torch.autograd.grad((dense_out, dense_balance), leaves, (grad.float(), share))
    assert torch.equal(balance.counts, chosen)
    for got, want in zip((out, balance.loss, *found), (dense_out, dense_balance, *wanted)):
        assert (got.float() - want.float()).norm() <= TOLERANCE * want.float().norm()


def parse_args(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--tokens", type=int, default=129)
    parser.add_argument("--hidden", type=int, default=1024)
    parser.add_argument("--intermediate", type=int, default=512)
    parser.add_argument("--experts", type=int, default=8)
    parser.add_argument("--topk", type=int, default=3)
    parser.add_argument("--alignment", type=int, default=16)
    parser.add_argument("--steps", type=int, default=2)
    parser.add_argument("--train", action="store_true", help="the gradients instead of the layer in 8 bits")
    options = parser.parse_args(argv)
    for name in ("tokens", "hidden", "intermediate", "experts", "topk", "alignment", "steps"):
        if getattr(options, name) <= 0:
            parser.error(f"{name} must be positive")
    if options.hidden % 256 or options.intermediate % 16:
        parser.error("hidden must be a multiple of 256 and intermediate one of 16")
    if options.topk > options.experts:
        parser.error("topk must not exceed experts")
    return options


def run(options) -> dict:
    (train if options.train else serve)(options)
    torch.cuda.synchronize()
    return vars(options)


if __name__ == "__main__":
    print("NANO_EP_FP8_MOE_OK=" + json.dumps(run(parse_args())), flush=True)
