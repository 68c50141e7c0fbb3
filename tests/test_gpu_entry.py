"""The operators at an expert layer's entry on the GPU against their definitions in 64 bits."""

import math

import pytest
import torch

import entry_oracle as oracle
import nanoep_amd as ep

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
TYPES = [(BF16, BF16), (BF16, FP32), (FP32, FP32)]
LOWEST = torch.finfo(FP32).min


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def to(device, *tensors):
    return tuple(None if tensor is None else tensor.to(device) for tensor in tensors)


def same_bits(a, b):
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


# ------------------------------------------------------------------ norms


def make_norm(tokens, hidden, rows, parameters, seed, residual=True, offset=0.3):
    x = (3 * randn(seed, tokens, hidden) + offset).to(rows)
    other = randn(seed + 1, tokens, hidden).to(rows) if residual else None
    gamma = (1 + 0.2 * randn(seed + 2, hidden)).to(parameters)
    beta = (0.5 * randn(seed + 3, hidden)).to(parameters)
    return x, other, gamma, beta


def run_norm(kind, x, gamma, beta, residual, eps):
    if kind == "layer":
        return ep.layer_norm(x, gamma, beta, residual=residual, eps=eps)
    return ep.rms_norm(x, gamma, residual=residual, eps=eps)


def check_norm(device, kind, x, residual, gamma, beta, eps):
    beta = beta if kind == "layer" else None
    got = run_norm(kind, *to(device, x, gamma, beta, residual), eps)
    s = oracle.total_of(x, residual)
    y, mean, rstd = oracle.norm(s, gamma, beta, eps, kind == "layer")
    assert (got.residual is None) == (residual is None)
    if residual is not None:
        assert same_bits(got.residual.cpu(), s)
    oracle.check_rounded(got.normalized, *y, x.dtype)
    oracle.check_rounded(got.rstd, *rstd, FP32)
    assert (got.mean is None) == (kind == "rms")
    if kind == "layer":
        oracle.check_rounded(got.mean, *mean, FP32)
    return got


@pytest.mark.parametrize("hidden", [8, 64, 72, 256, 504, 512, 520, 1000, 1024, 1032, 2816, 7168, 8200, 16384])
@pytest.mark.parametrize("tokens", [1, 5, 1027])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,parameters", TYPES)
def test_norm(device, kind, tokens, hidden, rows, parameters):
    if tokens > 5 and hidden > 1032:
        tokens = 1024 if hidden == 2816 else 37
    print("norm", kind, tokens, hidden, rows, parameters, flush=True)
    x, residual, gamma, beta = make_norm(tokens, hidden, rows, parameters, hidden + tokens, residual=hidden % 16 == 8 or tokens == 1)
    check_norm(device, kind, x, residual, gamma, beta, 1e-5)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norm_options(device, kind):
    x, residual, gamma, beta = make_norm(7, 1024, BF16, BF16, 3)
    print("norm options", kind, flush=True)
    check_norm(device, kind, x, residual, gamma, None, 1e-5)
    check_norm(device, kind, x, None, gamma, beta, 0.0)
    check_norm(device, kind, x, None, gamma, None, 3.0)


@pytest.mark.parametrize("rows", [BF16, FP32])
def test_norm_of_rows_far_from_zero(device, rows):
    """A mean a thousand times the deviation: squares are of what is left of it."""
    x, _, gamma, beta = make_norm(9, 2048, rows, FP32, 5, residual=False, offset=3000.0)
    print("norm far from zero", rows, flush=True)
    check_norm(device, "layer", x, None, gamma, beta, 1e-5)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows", [BF16, FP32])
@pytest.mark.parametrize("power", [-58, -20, 20, 55])
def test_norm_of_very_small_and_very_large_rows(device, kind, rows, power):
    """As far as the squares are in fp32, a factor of all rows is one of nothing but the statistics and the gradient."""
    total, _, gamma, beta = make_norm(9, 520, rows, FP32, 6, residual=False)
    total = total * 2.0**power
    print("norm of scaled rows", kind, rows, power, flush=True)
    check_norm(device, kind, total, None, gamma, beta, 0.0)
    check_norm_backward(device, kind, randn(7, 9, 520).to(rows), total, gamma, None, eps=0.0)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("hidden", [512, 2816])
def test_norm_of_zeros_infinities_and_nan(device, kind, hidden):
    x, _, gamma, beta = make_norm(9, hidden, BF16, BF16, 7, residual=False)
    x[0] = 0
    x[2] = 5.0  # no deviation
    x[4, 300], x[6, 300] = math.inf, math.nan
    print("norm of zeros, infinities and nan", kind, hidden, flush=True)
    got = run_norm(kind, *to(device, x, gamma, beta if kind == "layer" else None, None), 1e-5)
    fine = [0, 1, 2, 3, 5, 7, 8]
    y, _, _ = oracle.norm(x[fine], gamma, beta if kind == "layer" else None, 1e-5, kind == "layer")
    oracle.check_rounded(got.normalized[fine], *y, BF16)
    broken = got.normalized[[4, 6]].cpu()
    assert broken[0, 300].isnan() and broken[1].isnan().all() and (broken[0].isnan().all() if kind == "layer" else True)
    g = randn(8, 9, hidden).to(BF16).to(device)
    if kind == "layer":
        grad_x, grad_gamma, _ = ep.layer_norm_backward(g, x.to(device), gamma.to(device), got.mean, got.rstd)
    else:
        grad_x, grad_gamma = ep.rms_norm_backward(g, x.to(device), gamma.to(device), got.rstd)
    assert grad_x[fine].isfinite().all() and not grad_x[[4, 6]].isfinite().all() and not grad_gamma.isfinite().all()


def check_norm_backward(device, kind, grad, total, gamma, grad_residual, eps=1e-5, **wanted):
    _, (mean, _), (rstd, _) = oracle.norm(total, gamma, None, eps, kind == "layer")
    mean, rstd = mean.float() if kind == "layer" else None, rstd.float()
    want = oracle.norm_backward(grad, total, gamma, mean, rstd, grad_residual)
    g, t, w, m, r, more = to(device, grad, total, gamma, mean, rstd, grad_residual)
    if kind == "layer":
        got = ep.layer_norm_backward(g, t, w, m, r, grad_residual=more, **wanted)
    else:
        got = (*ep.rms_norm_backward(g, t, w, r, grad_residual=more, **wanted), None)
    types = (total.dtype, gamma.dtype, gamma.dtype)
    asked = (wanted.get("input", True), wanted.get("parameters", True), wanted.get("parameters", True) and kind == "layer")
    for found, (value, slack), dtype, ask in zip(got, want, types, asked):
        assert (found is not None) == ask
        if ask:
            oracle.check_rounded(found, value, slack, dtype)


@pytest.mark.parametrize("hidden", [8, 64, 72, 256, 504, 512, 520, 1000, 1024, 1032, 2816, 7168, 8200, 16384])
@pytest.mark.parametrize("tokens", [1, 5, 1027])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,parameters", TYPES)
def test_norm_backward(device, kind, tokens, hidden, rows, parameters):
    if tokens > 5 and hidden > 1032:
        tokens = 1024 if hidden == 2816 else 37
    print("norm backward", kind, tokens, hidden, rows, parameters, flush=True)
    total, grad_residual, gamma, _ = make_norm(tokens, hidden, rows, parameters, hidden, residual=hidden % 16 == 8 or tokens == 1)
    check_norm_backward(device, kind, randn(tokens, tokens, hidden).to(rows), total, gamma, grad_residual)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("tokens,hidden", [(513, 1152), (1025, 640), (4097, 136), (9000, 64)])
def test_norm_backward_of_several_rows_a_workgroup(device, kind, tokens, hidden):
    print("norm backward", kind, tokens, hidden, flush=True)
    total, grad_residual, gamma, _ = make_norm(tokens, hidden, BF16, FP32, hidden)
    check_norm_backward(device, kind, randn(tokens, tokens, hidden).to(BF16), total, gamma, grad_residual)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("wanted", [{"input": False}, {"parameters": False}])
def test_norm_backward_gives_what_is_asked_for(device, kind, wanted):
    total, grad_residual, gamma, _ = make_norm(70, 1024, BF16, BF16, 4)
    print("norm backward", kind, wanted, flush=True)
    check_norm_backward(device, kind, randn(5, 70, 1024).to(BF16), total, gamma, grad_residual, **wanted)


def test_norm_of_no_tokens(device):
    empty, gamma = torch.empty(0, 256, dtype=BF16, device=device), torch.ones(256, device=device)
    got = ep.layer_norm(empty, gamma, gamma, residual=empty)
    assert got.normalized.shape == got.residual.shape == (0, 256) and got.mean.shape == got.rstd.shape == (0,)
    grad_x, grad_gamma, grad_beta = ep.layer_norm_backward(empty, empty, gamma, got.mean, got.rstd)
    assert grad_x.shape == (0, 256) and not grad_gamma.any() and not grad_beta.any()
    grad_x, grad_gamma = ep.rms_norm_backward(empty, empty, gamma, got.rstd)
    assert grad_x.shape == (0, 256) and not grad_gamma.any()


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_the_norms_gradient_is_the_difference(device, kind):
    """(f(x + d) - f(x - d)) / 2 in 64 bits along random directions, against the gradient in fp32."""
    tokens, hidden, eps = 6, 320, 1e-5
    x, residual, gamma, beta = make_norm(tokens, hidden, FP32, FP32, 21)
    grad, grad_residual = randn(22, tokens, hidden), randn(23, tokens, hidden)
    leaves = [tensor.to(device).requires_grad_() for tensor in (x, residual, gamma, beta)]
    result = run_norm(kind, leaves[0], leaves[2], leaves[3], leaves[1], eps)
    inputs = leaves if kind == "layer" else leaves[:3]
    found = torch.autograd.grad((result.normalized, result.residual), inputs, (grad.to(device), grad_residual.to(device)))

    def value(x, residual, gamma, beta):
        s = x + residual
        c = s - s.mean(1, keepdim=True) if kind == "layer" else s
        y = c * ((c * c).mean(1, keepdim=True) + eps).rsqrt() * gamma + (beta if kind == "layer" else 0)
        return (y * grad.double()).sum() + (s * grad_residual.double()).sum()

    base = [tensor.double() for tensor in (x, residual, gamma, beta)]
    for which, gradient in enumerate(found):
        for seed in range(3):
            step = [torch.zeros_like(tensor) for tensor in base]
            step[which] = 1e-5 * randn(seed, *base[which].shape).double()
            change = (value(*(a + b for a, b in zip(base, step))) - value(*(a - b for a, b in zip(base, step)))) / 2
            terms = gradient.cpu().double() * step[which]
            # the gradient's own rounding, and the step's third order
            assert abs(change - terms.sum()) <= 400 * oracle.FP32 * terms.abs().sum() + 1e-9 * step[which].abs().sum()


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_autograd_through_norms(device, kind):
    tokens, hidden = 33, 512
    x, residual, gamma, beta = make_norm(tokens, hidden, BF16, BF16, 31)
    grad, grad_residual = randn(32, tokens, hidden).to(BF16), randn(33, tokens, hidden).to(BF16)
    x, residual, gamma, beta, grad, grad_residual = to(device, x, residual, gamma, beta, grad, grad_residual)
    every = [x, residual, gamma] + ([beta] if kind == "layer" else [])
    for wanted in range(1, 1 << len(every)):
        leaves = [tensor.detach().requires_grad_(bool(wanted >> i & 1)) for i, tensor in enumerate(every)]
        result = run_norm(kind, leaves[0], leaves[2], leaves[3] if kind == "layer" else None, leaves[1], 1e-5)
        assert not result.rstd.requires_grad
        asked = [leaf for leaf in leaves if leaf.requires_grad]
        found = dict(zip(map(id, asked), torch.autograd.grad((result.normalized, result.residual), asked, (grad, grad_residual))
                         if leaves[0].requires_grad or leaves[1].requires_grad else torch.autograd.grad(result.normalized, asked, grad)))
        plain = run_norm(kind, x, gamma, beta if kind == "layer" else None, residual, 1e-5)
        if kind == "layer":
            want = ep.layer_norm_backward(grad, plain.residual, gamma, plain.mean, plain.rstd, grad_residual=grad_residual)
        else:
            want = ep.rms_norm_backward(grad, plain.residual, gamma, plain.rstd, grad_residual=grad_residual)
        for leaf, value in zip(leaves, (want[0], want[0], *want[1:])):
            if leaf.requires_grad:
                assert same_bits(found[id(leaf)], value)


def test_autograd_of_one_of_a_norms_outputs(device):
    x, residual, gamma, _ = to(device, *make_norm(12, 256, BF16, FP32, 41))
    grad = randn(42, 12, 256).to(BF16).to(device)
    x.requires_grad_()
    gamma.requires_grad_()
    only_sum = ep.rms_norm(x, gamma, residual=residual).residual
    found = torch.autograd.grad(only_sum, (x, gamma), grad, allow_unused=True)
    assert same_bits(found[0], grad) and (found[1] is None or not found[1].any())
    only_norm = ep.rms_norm(x, gamma, residual=residual)
    (found,) = torch.autograd.grad(only_norm.normalized, x, grad)
    want, _ = ep.rms_norm_backward(grad, only_norm.residual.detach(), gamma.detach(), only_norm.rstd)
    assert same_bits(found, want)


def test_norm_gradients_that_arrive_in_other_layouts(device):
    """Expanded, transposed, and off a 16-byte boundary."""
    x, _, gamma, beta = to(device, *make_norm(16, 256, BF16, BF16, 43, residual=False))
    x.requires_grad_()
    first = ep.layer_norm(x, gamma, beta)
    (found,) = torch.autograd.grad(first.normalized.sum(), x)
    ones = torch.ones(16, 256, dtype=BF16, device=device)
    want, _, _ = ep.layer_norm_backward(ones, x.detach(), gamma, first.mean, first.rstd)
    assert same_bits(found, want)
    factor = randn(44, 256, 16).to(BF16).to(device)
    (found,) = torch.autograd.grad(ep.layer_norm(x, gamma, beta).normalized, x, factor.T)
    want, _, _ = ep.layer_norm_backward(factor.T.contiguous(), x.detach(), gamma, first.mean, first.rstd)
    assert same_bits(found, want)
    flat = torch.zeros(3 + 16 * 256, dtype=BF16, device=device)
    off = flat[3:].view(16, 256).copy_(factor.T)
    (found,) = torch.autograd.grad(ep.layer_norm(x, gamma, beta).normalized, x, off)
    assert same_bits(found, want)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("tokens,hidden,rows,parameters,residual", [(8200, 8192, BF16, BF16, True), (7000, 8200, BF16, FP32, True), (30000, 1032, FP32, FP32, True),
                                                                    (1600, 16384, FP32, FP32, True), (250000, 504, BF16, FP32, False)])
def test_norm_of_more_rows_than_the_last_level_cache_holds(device, kind, tokens, hidden, rows, parameters, residual):
    generator = torch.Generator(device=device).manual_seed(hidden)
    x = (3 * torch.randn(tokens, hidden, device=device, generator=generator) + 0.3).to(rows)
    other = torch.randn(tokens, hidden, device=device, generator=generator).to(rows) if residual else None
    gamma = (1 + 0.2 * torch.randn(hidden, device=device, generator=generator)).to(parameters)
    beta = (0.5 * torch.randn(hidden, device=device, generator=generator)).to(parameters) if kind == "layer" else None
    print("norm, many rows", kind, tokens, hidden, rows, flush=True)
    got = run_norm(kind, x, gamma, beta, other, 1e-5)
    some = torch.cat([torch.arange(5), torch.arange(tokens // 2, tokens // 2 + 40), torch.arange(tokens - 19, tokens)])
    s = oracle.total_of(x[some].cpu(), None if other is None else other[some].cpu())
    if residual:
        assert same_bits(got.residual[some].cpu(), s) and same_bits(got.residual, (x.float() + other.float()).to(rows))
    y, mean, rstd = oracle.norm(s, gamma.cpu(), None if beta is None else beta.cpu(), 1e-5, kind == "layer")
    oracle.check_rounded(got.normalized[some], *y, rows)
    oracle.check_rounded(got.rstd[some], *rstd, FP32)
    # all of them are what they are in a smaller batch
    for at in range(0, tokens, 1000):
        part = run_norm(kind, x[at : at + 1000], gamma, beta, None if other is None else other[at : at + 1000], 1e-5)
        assert same_bits(got.normalized[at : at + 1000], part.normalized) and same_bits(got.rstd[at : at + 1000], part.rstd)


def test_norm_rows_beyond_32_bit_offsets(device):
    tokens, hidden = 330_000, 7168
    gamma = torch.ones(hidden, dtype=BF16, device=device)
    x = torch.empty(tokens, hidden, dtype=BF16, device=device)
    part = randn(51, 1000, hidden).to(BF16).to(device)
    for at in range(0, tokens, 1000):
        x[at : at + 1000] = part
    print("norm beyond 32 bits", tokens, hidden, flush=True)
    whole = ep.rms_norm(x, gamma, residual=x)
    want = ep.rms_norm(part, gamma, residual=part)
    for at in (0, 150_000, 299_000, 329_000):
        assert same_bits(whole.normalized[at : at + 1000], want.normalized) and same_bits(whole.rstd[at : at + 1000], want.rstd)
        assert same_bits(whole.residual[at : at + 1000], want.residual)
    grad_x, _ = ep.rms_norm_backward(x, whole.residual, gamma, whole.rstd)
    want_x, _ = ep.rms_norm_backward(part, want.residual, gamma, want.rstd)
    for at in (0, 299_000, 329_000):
        assert same_bits(grad_x[at : at + 1000], want_x)


# ------------------------------------------------------------------ router

SCORINGS = ["softmax", "sigmoid"]
EXPERTS = [1, 2, 7, 8, 16, 31, 60, 64, 65, 128, 200, 256, 257, 512, 1000, 1024, 2048, 3839, 4096]


def check_route(device, logits, topk, *, scoring="softmax", bias=None, mask=None, groups=1, topk_groups=1, normalize=True, scale=1.0, on=None):
    got = ep.route_topk(logits.to(device) if on is None else on, topk, scoring=scoring, bias=None if bias is None else bias.to(device),
                        mask=None if mask is None else mask.to(device), groups=groups, topk_groups=topk_groups, normalize=normalize, scale=scale)
    ids = oracle.choose(logits, topk, scoring, bias, mask, groups, topk_groups)
    assert got.ids.dtype == torch.int64 and torch.equal(got.ids.cpu(), ids)
    weights, slack = oracle.weigh(logits, ids, scoring, normalize, scale)
    oracle.check_rounded(got.weights, weights, slack, FP32)
    assert not got.weights.cpu()[ids < 0].any()
    return got


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("biased", [False, True])
def test_route(device, experts, scoring, normalize, biased):
    for tokens, topk, dtype in ((1, min(8, experts), FP32), (67, min(experts, 32), BF16), (300, (experts + 7) // 8 % 9 + 1, FP32)):
        topk = min(topk, experts)
        print("route", tokens, experts, topk, scoring, normalize, biased, dtype, flush=True)
        logits = (2 * randn(experts + tokens, tokens, experts)).to(dtype)
        bias = (20 * randn(3, experts)).round() / 100 if biased else None
        mask = torch.arange(tokens) % 7 != 3 if tokens > 1 else None
        check_route(device, logits, topk, scoring=scoring, bias=bias, mask=mask, normalize=normalize, scale=1.0 if normalize else 2.5)


@pytest.mark.parametrize("experts,groups,topk_groups,topk", [(8, 8, 2, 2), (8, 2, 1, 4), (60, 3, 2, 6), (64, 64, 5, 5), (200, 8, 3, 8), (256, 8, 4, 8),
                                                            (256, 16, 1, 16), (255, 5, 5, 9), (320, 5, 2, 8), (1000, 40, 7, 10), (2048, 32, 4, 32), (4096, 64, 8, 8), (3840, 3, 1, 32)])
@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("biased", [False, True])
def test_route_within_groups(device, experts, groups, topk_groups, topk, scoring, biased):
    for tokens, dtype in ((1, FP32), (130, BF16), (77, FP32)):
        print("route within groups", tokens, experts, groups, topk_groups, topk, scoring, biased, flush=True)
        logits = (2 * randn(experts + tokens, tokens, experts)).to(dtype)
        logits[:, ::5] -= 1.5
        if tokens > 1:
            logits[3, experts // 2 :] = -math.inf
            logits[5, : experts // groups] = -math.inf
            logits[6] = -math.inf
            logits[7, 1:] = -math.inf
        check_route(device, logits, topk, scoring=scoring, bias=0.1 * randn(4, experts) if biased else None, groups=groups, topk_groups=topk_groups,
                    normalize=tokens != 77, scale=2.5)


@pytest.mark.parametrize("experts", [8, 60, 64, 128, 256, 1000])
@pytest.mark.parametrize("biased", [False, True])
def test_ties_go_to_the_lowest_index(device, experts, biased):
    generator = torch.Generator().manual_seed(experts)
    logits = torch.randint(-1, 2, (200, experts), generator=generator).float()
    logits[1] = 0.0
    logits[2, ::2] = -0.0
    logits[2, 1::2] = 0.0
    bias = torch.randint(0, 2, (experts,), generator=generator).float() * 0.25 if biased else None
    for topk in (1, 4, 8):
        for dtype in (FP32, BF16):
            print("ties", experts, topk, biased, dtype, flush=True)
            for scoring in SCORINGS:
                check_route(device, logits.to(dtype), topk, scoring=scoring, bias=bias)
                if experts % 4 == 0:
                    check_route(device, logits.to(dtype), min(topk, experts // 2), scoring=scoring, bias=bias, groups=4, topk_groups=2)


@pytest.mark.parametrize("scoring", SCORINGS)
def test_route_of_long_batches(device, scoring):
    """More tokens than a device's wavefronts take one each of: fewer lanes a token."""
    for experts, topk, groups, topk_groups in ((3, 2, 1, 1), (8, 6, 4, 3), (16, 3, 1, 1), (31, 12, 1, 1), (32, 4, 8, 4), (60, 6, 3, 2), (64, 16, 1, 1), (100, 4, 5, 2), (128, 8, 1, 1),
                                               (200, 16, 8, 3), (256, 8, 8, 4), (300, 20, 1, 1), (512, 6, 16, 5)):
        tokens = 8200 + experts
        print("route, long", tokens, experts, topk, scoring, flush=True)
        logits = 2 * randn(experts, tokens, experts)
        logits[:200] = logits[:200].round()  # equal ones
        logits[300, 1:] = -math.inf
        logits[301:308] = 0.5  # all of them
        logits[308] = -math.inf
        mask = torch.arange(tokens) < tokens - 5
        bias = (20 * randn(experts + 1, experts)).round() / 100
        grad = randn(9, tokens, topk)
        for normalize, dtype in ((True, BF16), (False, FP32)):
            got = check_route(device, logits.to(dtype), topk, scoring=scoring, normalize=normalize, mask=mask)
            check_route(device, logits.to(dtype), topk, scoring=scoring, normalize=normalize, bias=bias, groups=groups, topk_groups=topk_groups)
            check_route(device, logits.to(dtype), topk, scoring=scoring, normalize=normalize, groups=groups, topk_groups=topk_groups)
            check_route(device, logits.to(dtype), topk, scoring=scoring, normalize=normalize, bias=torch.zeros(experts))
            logits[308] = 0.0
            found = ep.route_topk_backward(grad.to(device), logits.to(dtype).to(device), got.ids, scoring=scoring, normalize=normalize)
            oracle.check_rounded(found, *oracle.weigh_backward(grad, logits.to(dtype), got.ids.cpu(), scoring, normalize, 1.0), dtype)
            logits[308] = -math.inf


@pytest.mark.parametrize("scoring", SCORINGS)
def test_values_that_fp32_cannot_tell_apart(device, scoring):
    """Neighbouring logits: their scores are one value in fp32, and their biased scores too, but not in 64 bits."""
    tokens, experts = 64, 32
    logits = torch.full((tokens, experts), 1.0)
    for t in range(tokens):
        for e in range(experts):
            logits[t, e] = 1.0 + 2.0**-23 * ((e * 7 + t) % experts)
    print("neighbours", scoring, flush=True)
    check_route(device, logits, 8, scoring=scoring)
    check_route(device, logits, 8, scoring=scoring, bias=torch.full((experts,), 0.125))
    check_route(device, logits, 8, scoring=scoring, groups=4, topk_groups=2)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,size", [(8, 32), (16, 1), (16, 2), (12, 5), (64, 4), (4, 200)])
def test_groups_that_fp32_cannot_tell_apart(device, scoring, biased, groups, size):
    """Every group's largest value is a neighbour of the others' largest, some are equal; their second ones are the same."""
    tokens, experts = 70, groups * size
    logits = randn(67, tokens, groups, size).clamp(max=0.5) - 2.0
    step = torch.stack([torch.randperm(groups, generator=torch.Generator().manual_seed(t)) for t in range(tokens)])
    step[1::3] //= 2  # equal ones
    logits[:, :, size // 2] = 1.0 + 2.0**-23 * step
    if size > 2:
        logits[:, :, size - 1] = 0.75
        logits[5] = 1.0  # all of them, more than a list holds
        logits[6, : groups // 2] = 1.0 + 2.0**-23 * step[6, : groups // 2, None]
        logits[7, 1:3] = -math.inf
    logits = logits.reshape(tokens, experts)
    bias = torch.full((experts,), 0.125) if biased else None
    print("groups, neighbours", scoring, biased, groups, size, flush=True)
    for kept in (1, groups // 2, groups - 1):
        topk = min(8, kept * size)
        check_route(device, logits, topk, scoring=scoring, bias=bias, groups=groups, topk_groups=kept)
        check_route(device, logits[:1], topk, scoring=scoring, bias=bias, groups=groups, topk_groups=kept)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("experts", [6, 64, 256])
def test_route_of_masked_and_extreme_logits(device, scoring, normalize, biased, experts):
    logits = randn(61, 12, experts)
    logits[0] = -math.inf  # nothing is left
    logits[1, 2:] = -math.inf  # fewer than topk
    logits[2, :-1] = -math.inf  # only the last
    logits[3] = LOWEST  # masked with the type's lowest: values like others
    logits[4, 1:] = LOWEST
    logits[5] *= 1e4
    logits[6] = -200.0 - torch.arange(experts)  # sigmoids that fp32 cannot hold
    logits[7] = 80.0 + torch.arange(experts)
    logits[8, 0] = 1e30
    logits[9] -= 90.0
    bias = 0.01 * randn(62, experts) if biased else None
    print("extreme logits", scoring, normalize, biased, experts, flush=True)
    check_route(device, logits, 4, scoring=scoring, bias=bias, normalize=normalize)
    if biased:
        bias[:2] = -math.inf  # experts that are switched off
        check_route(device, logits, 4, scoring=scoring, bias=bias, normalize=normalize)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("biased", [False, True])
def test_route_of_nan_and_infinity(device, scoring, biased):
    experts, topk = 60, 6
    logits = randn(63, 6, experts)
    logits[1, 17] = math.nan
    logits[2, 40] = math.inf
    logits[3] = math.nan
    logits[4, [3, 9]] = math.nan
    bias = 0.01 * randn(64, experts) if biased else None
    for normalize in (True, False):
        print("nan", scoring, biased, normalize, flush=True)
        got = ep.route_topk(logits.to(device), topk, scoring=scoring, bias=None if bias is None else bias.to(device), normalize=normalize)
        ids, weights = got.ids.cpu(), got.weights.cpu()
        for row in ids:
            assert len(set(row.tolist())) == topk and 0 <= int(row.min()) and int(row.max()) < experts
        fine = [0, 5]
        assert torch.equal(ids[fine], oracle.choose(logits[fine], topk, scoring, bias)) and weights[fine].isfinite().all()
        if not (biased and scoring == "softmax"):  # (a softmax with a NaN is nothing but)
            assert ids[1, 0] == 17 and ids[2, 0] == 40 and ids[4, :2].tolist() == [3, 9]
        if normalize or scoring == "softmax":
            assert weights[[1, 3, 4]].isnan().any(1).all()
        found = ep.route_topk_backward(torch.ones(6, topk, device=device), logits.to(device), got.ids, scoring=scoring, normalize=normalize)
        assert found[fine].isfinite().all()


def test_route_reads_rows_any_distance_apart(device):
    wide = randn(65, 90, 300).to(device)
    for columns, dtype in ((slice(0, 256), FP32), (slice(4, 260), FP32), (slice(3, 259), BF16), (slice(8, 136), BF16), (slice(1, 61), FP32)):
        part = wide.to(dtype)[:, columns]
        print("strides", columns, dtype, flush=True)
        check_route(device, part.cpu(), 8, on=part)
        check_route(device, part.cpu(), 4, on=part, groups=4, topk_groups=2)
        grad = randn(66, 90, 8)
        ids = oracle.choose(part.cpu(), 8, "softmax")
        found = ep.route_topk_backward(grad.to(device), part, ids.to(device), normalize=False)
        oracle.check_rounded(found, *oracle.weigh_backward(grad, part.cpu(), ids, "softmax", False, 1.0), dtype)
    one = wide[:1, :64]
    assert torch.equal(ep.route_topk(one, 4).ids, ep.route_topk(one.contiguous(), 4).ids)


def test_route_of_no_tokens(device):
    empty = torch.empty(0, 64, device=device)
    got = ep.route_topk(empty, 8)
    assert got.ids.shape == got.weights.shape == (0, 8) and got.ids.dtype == torch.int64
    assert ep.route_topk_backward(got.weights, empty, got.ids).shape == (0, 64)


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("normalize", [True, False])
def test_route_backward(device, experts, scoring, normalize):
    for tokens, topk, dtype in ((1, min(8, experts), FP32), (67, 32, BF16), (300, (experts + 7) // 8 % 9 + 1, FP32)):
        print("route backward", tokens, experts, topk, scoring, normalize, dtype, flush=True)
        logits = (2 * randn(experts + tokens, tokens, experts)).to(dtype)
        # any choices, among them masked ones, ones that are no expert, and the same one twice
        ids = torch.randint(-2, experts + 2, (tokens, topk), generator=torch.Generator().manual_seed(experts))
        if tokens > 5:
            ids[4] = -1
        grad = randn(7, tokens, topk)
        found = ep.route_topk_backward(grad.to(device), logits.to(device), ids.to(device), scoring=scoring, normalize=normalize, scale=2.5)
        oracle.check_rounded(found, *oracle.weigh_backward(grad, logits, ids, scoring, normalize, 2.5), dtype)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("normalize", [True, False])
def test_route_backward_of_masked_and_extreme_logits(device, scoring, normalize):
    """Choices of experts that could not have been chosen among them, and gradients of masked choices that are not looked at."""
    tokens, experts, topk = 8, 40, 4
    logits, grad = randn(73, tokens, experts), randn(74, tokens, topk)
    ids = torch.arange(topk).repeat(tokens, 1) * 9
    logits[0] = -math.inf
    logits[0, 39] = 1.0
    logits[1, :20] = -math.inf
    logits[2] = LOWEST
    logits[3, 9] = LOWEST
    logits[4] = -300.0 - torch.arange(experts)
    logits[5] = 90.0 + torch.arange(experts)
    ids[6, 1], ids[6, 3] = -1, experts
    grad[6, 1], grad[6, 3] = math.nan, math.inf
    print("route backward, extreme", scoring, normalize, flush=True)
    found = ep.route_topk_backward(grad.to(device), logits.to(device), ids.to(device), scoring=scoring, normalize=normalize)
    oracle.check_rounded(found, *oracle.weigh_backward(grad, logits, ids, scoring, normalize, 1.0), FP32)
    assert found.isfinite().all()


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("normalize", [True, False])
def test_the_routers_gradient_is_the_difference(device, scoring, normalize):
    tokens, experts, topk = 9, 40, 5
    logits, grad = randn(71, tokens, experts), randn(72, tokens, topk)
    leaf = logits.to(device).requires_grad_()
    routing = ep.route_topk(leaf, topk, scoring=scoring, normalize=normalize, scale=1.5)
    assert not routing.ids.requires_grad
    (found,) = torch.autograd.grad(routing.weights, leaf, grad.to(device))
    ids = routing.ids.cpu()
    for seed in range(4):
        step = 1e-5 * randn(seed, tokens, experts).double()
        plus, _ = oracle.weigh(logits.double() + step, ids, scoring, normalize, 1.5)
        minus, _ = oracle.weigh(logits.double() - step, ids, scoring, normalize, 1.5)
        change = ((plus - minus) / 2 * grad.double()).sum()
        terms = found.cpu().double() * step
        assert abs(change - terms.sum()) <= 400 * oracle.FP32 * terms.abs().sum() + 1e-9 * step.abs().sum()


# ------------------------------------------------------------------ balance


def make_balance(tokens, experts, topk, seed, dtype=FP32):
    logits = (1.5 * randn(seed, tokens, experts) + randn(seed + 1, experts)).to(dtype)
    ids = logits.float().topk(min(topk, experts), dim=1).indices
    drop = torch.rand(ids.shape, generator=torch.Generator().manual_seed(seed + 2)) < 0.15
    ids = ids.masked_fill(drop, -1)
    ids[1::6] = -1
    return logits, ids


def check_balance(device, logits, ids, scoring, offsets=None, on=None):
    logits_on = logits.to(device) if on is None else on
    ids_on, offsets_on = ids.to(device), None if offsets is None else torch.tensor(offsets, device=device)
    grad = 0.5 + torch.rand(1 if offsets is None else len(offsets) - 1, generator=torch.Generator().manual_seed(1))
    got = ep.balance_loss(logits_on, ids_on, scoring=scoring, sequence_offsets=offsets_on)
    counts, tokens, (loss, loss_slack), (want, slack) = oracle.balance(logits, ids, scoring, offsets, grad)
    shape = () if offsets is None else (len(offsets) - 1,)
    assert got.loss.shape == got.tokens.shape == shape and got.counts.shape == (*shape, logits.shape[1])
    assert torch.equal(got.counts.cpu().view_as(counts), counts) and torch.equal(got.tokens.cpu().view_as(tokens), tokens)
    oracle.check_rounded(got.loss.view(-1), loss, loss_slack, FP32)
    found = ep.balance_loss_backward(grad.to(device).view(shape), logits_on, ids_on, got.counts, got.tokens, scoring=scoring, sequence_offsets=offsets_on)
    oracle.check_rounded(found, want, slack, logits.dtype)
    return got, found


@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("scoring", SCORINGS)
def test_balance_loss(device, experts, scoring):
    for tokens, topk, dtype in ((1, 8, FP32), (3, 2, BF16), (67, 32, BF16), (700, (experts + 7) // 8 % 9 + 1, FP32)):
        print("balance", tokens, experts, topk, scoring, dtype, flush=True)
        check_balance(device, *make_balance(tokens, experts, topk, experts + tokens, dtype), scoring)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("experts", [8, 60, 256, 1000])
@pytest.mark.parametrize("offsets", [[0, 500], [0, 0, 1, 3, 3, 130, 490], [0, 250, 500], [0, 64, 128, 500], [2, 6, 200], [0, 0, 0], list(range(0, 501, 4))])
def test_balance_loss_of_sequences(device, offsets, experts, scoring):
    logits, ids = make_balance(500, experts, 6, experts)
    ids[3:130] = -1  # (a sequence of padding)
    print("balance of sequences", len(offsets), experts, scoring, flush=True)
    check_balance(device, logits, ids, scoring, offsets)


@pytest.mark.parametrize("scoring", SCORINGS)
def test_balance_loss_of_many_short_sequences(device, scoring):
    """Some empty, most of a few tokens, more than are searched at once."""
    generator = torch.Generator().manual_seed(89)
    for tokens, sequences, experts, topk in ((5000, 4500, 24, 3), (9000, 300, 60, 12), (700, 66, 130, 20)):
        lengths = torch.randint(0, 2 * tokens // sequences + 1, (sequences,), generator=generator)
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]).clamp(max=tokens - 3).tolist()
        print("balance, short sequences", tokens, sequences, experts, topk, scoring, flush=True)
        logits, ids = make_balance(tokens, experts, topk, experts)
        check_balance(device, logits, ids, scoring, offsets)


def test_balance_loss_of_long_batches(device):
    for tokens, experts, topk in ((20000, 16, 4), (30001, 60, 2)):
        print("balance, long", tokens, experts, flush=True)
        logits, ids = make_balance(tokens, experts, topk, experts)
        check_balance(device, logits, ids, "softmax")
        check_balance(device, logits, ids, "sigmoid", [0, 7, 9000, 9001, tokens - 5])


@pytest.mark.parametrize("scoring", SCORINGS)
def test_balance_loss_does_not_look_at_padding(device, scoring):
    logits, ids = make_balance(300, 60, 6, 81)
    ids[200:] = -1
    ids[100:110] = 60  # no expert
    ids[110:120] = -7
    broken = logits.clone()
    broken[(ids < 0).all(1) | (ids >= 60).all(1)] = math.nan
    want, want_grad = check_balance(device, logits, ids, scoring)
    got, grad = check_balance(device, broken, ids, scoring)
    assert same_bits(got.loss, want.loss) and same_bits(grad, want_grad)


@pytest.mark.parametrize("scoring", SCORINGS)
def test_balance_loss_of_masked_and_extreme_logits(device, scoring):
    logits, ids = make_balance(64, 60, 4, 83)
    ids = ids.clamp(min=0)
    logits[0, 10:] = -math.inf
    logits[1] = -math.inf  # a token whose choices have no share
    logits[2] = LOWEST
    logits[3, 1:] = LOWEST
    logits[4] = -300.0 - torch.arange(60)
    logits[5] = 90.0 + torch.arange(60)
    logits[6] *= 1e4
    print("balance, extreme", scoring, flush=True)
    got, grad = check_balance(device, logits, ids, scoring)
    assert got.loss.isfinite() and grad.isfinite().all()
    logits[7, 3] = math.nan
    got, grad = ep.balance_loss(logits.to(device), ids.to(device), scoring=scoring), None
    assert got.loss.isnan()
    grad = ep.balance_loss_backward(torch.ones((), device=device), logits.to(device), ids.to(device), got.counts, got.tokens, scoring=scoring)
    assert grad[7].isnan().any() and grad[8:].isfinite().all() and grad[:7].isfinite().all()


def test_balance_loss_of_an_even_batch_is_one(device):
    tokens, experts = 256, 64
    ids = torch.arange(tokens * 4).view(tokens, 4) % experts
    for scoring in SCORINGS:
        got = ep.balance_loss(torch.zeros(tokens, experts, device=device), ids.to(device), scoring=scoring)
        assert abs(float(got.loss) - 1.0) <= 64 * oracle.FP32 and (got.counts == tokens * 4 // experts).all() and got.tokens == tokens


def test_balance_loss_of_one_sequence_without_tokens(device):
    """The batch's tokens are behind it; nothing that lay in the outputs' memory stays."""
    for tokens, experts in ((1, 1045), (3, 64), (40, 8), (500, 16), (3000, 256)):
        logits, ids = make_balance(tokens, experts, 4, 90)
        for offsets in ([0, 0], [0, tokens // 2], [0, 0, 0]):
            print("balance, one sequence", tokens, experts, offsets, flush=True)
            filled = [torch.full((size,), 77, dtype=torch.int64, device=device) for size in (1, 2, experts, 2 * experts) for _ in range(8)]
            del filled
            check_balance(device, logits, ids, "softmax", offsets)


def test_balance_loss_of_nothing(device):
    empty, ids = torch.empty(0, 8, device=device), torch.empty(0, 2, dtype=torch.int64, device=device)
    got = ep.balance_loss(empty, ids)
    assert got.loss == 0 and not got.counts.any() and got.tokens == 0
    assert ep.balance_loss_backward(got.loss, empty, ids, got.counts, got.tokens).shape == (0, 8)
    got = ep.balance_loss(empty, ids, sequence_offsets=torch.zeros(4, dtype=torch.int64, device=device))
    assert got.loss.tolist() == [0, 0, 0] and got.counts.shape == (3, 8)
    logits, ids = torch.randn(5, 8, device=device), torch.full((5, 2), -1, device=device)
    got = ep.balance_loss(logits, ids)
    assert got.loss == 0 and not ep.balance_loss_backward(got.loss + 1, logits, ids, got.counts, got.tokens).any()


@pytest.mark.parametrize("scoring", SCORINGS)
def test_the_balance_losses_gradient_is_the_difference(device, scoring):
    logits, ids = make_balance(60, 24, 3, 85)
    offsets = [0, 20, 50]
    leaf = logits.to(device).requires_grad_()
    result = ep.balance_loss(leaf, ids.to(device), scoring=scoring, sequence_offsets=torch.tensor(offsets, device=device))
    assert not result.counts.requires_grad and not result.tokens.requires_grad
    grad = torch.tensor([0.7, 1.9])
    (found,) = torch.autograd.grad(result.loss, leaf, grad.to(device))
    for seed in range(4):
        step = 1e-5 * randn(seed, *logits.shape).double()
        plus = oracle.balance(logits.double() + step, ids, scoring, offsets)[2][0]
        minus = oracle.balance(logits.double() - step, ids, scoring, offsets)[2][0]
        change = ((plus - minus) / 2 * grad.double()).sum()
        terms = found.cpu().double() * step
        assert abs(change - terms.sum()) <= 400 * oracle.FP32 * terms.abs().sum() + 1e-9 * step.abs().sum()


def test_balance_loss_stays_within_the_batch_whatever_the_offsets_say(device):
    logits, ids = make_balance(40, 24, 3, 87)
    for offsets in ([-5, 20, 60], [30, 10, 5], [0, 1 << 40], [-(1 << 40), 1 << 40], [50, 60]):
        print("offsets", offsets, flush=True)
        offsets = torch.tensor(offsets, device=device)
        got = ep.balance_loss(logits.to(device), ids.to(device), sequence_offsets=offsets)
        ep.balance_loss_backward(torch.ones_like(got.loss), logits.to(device), ids.to(device), got.counts, got.tokens, sequence_offsets=offsets)
    torch.cuda.synchronize()


def test_logits_beyond_32_bit_offsets(device):
    tokens, experts, topk = (1 << 25) + 3, 72, 2
    part = randn(91, 4096, experts).to(device)
    logits = torch.empty(tokens, experts, device=device)
    for at in range(0, tokens, 4096):
        logits[at : at + 4096] = part[: tokens - at]
    print("logits beyond 32 bits", tokens, experts, flush=True)
    whole, want = ep.route_topk(logits, topk), ep.route_topk(part, topk)
    last = (tokens - 1) // 4096 * 4096
    for at in (0, 1 << 24, last - 4096):
        assert torch.equal(whole.ids[at : at + 4096], want.ids) and same_bits(whole.weights[at : at + 4096], want.weights)
    assert torch.equal(whole.ids[last:], want.ids[: tokens - last])
    grad = torch.randn(4096, topk, device=device)
    wide = torch.empty(tokens, topk, device=device)
    for at in range(0, tokens, 4096):
        wide[at : at + 4096] = grad[: tokens - at]
    found = ep.route_topk_backward(wide, logits, whole.ids)
    assert same_bits(found[last - 4096 : last], ep.route_topk_backward(grad, part, want.ids))
    del found
    got = ep.balance_loss(logits, whole.ids)
    base = ep.balance_loss(part, want.ids)
    assert got.tokens == tokens and torch.equal(got.counts, base.counts * (tokens // 4096) + torch.bincount(want.ids[: tokens % 4096].reshape(-1), minlength=experts))
    found = ep.balance_loss_backward(torch.ones((), device=device), logits, whole.ids, got.counts, got.tokens)
    assert same_bits(found[last - 4096 : last], found[:4096]) and found[last:].any()


# ------------------------------------------------------------------ together


def test_entry_runs_on_the_current_stream(device):
    x, residual, gamma, beta = to(device, *make_norm(64, 512, BF16, BF16, 95))
    router = randn(96, 512, 32).to(device)
    want = ep.layer_norm(x, gamma, beta, residual=residual)
    want_routing = ep.route_topk(want.normalized.float() @ router, 4)
    want_balance = ep.balance_loss(want.normalized.float() @ router, want_routing.ids)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        later = torch.empty_like(x)
        torch.cuda._sleep(20_000_000)
        later.copy_(x)
        got = ep.layer_norm(later, gamma, beta, residual=residual)
        logits = got.normalized.float() @ router
        routing = ep.route_topk(logits, 4)
        balance = ep.balance_loss(logits, routing.ids)
        event = torch.cuda.Event()
        event.record()
    event.synchronize()
    assert same_bits(got.normalized, want.normalized) and torch.equal(routing.ids, want_routing.ids)
    assert same_bits(routing.weights, want_routing.weights) and same_bits(balance.loss, want_balance.loss)


def entry(x, residual, gamma, beta, logits, grad, grad_weights, offsets):
    normed = ep.layer_norm(x, gamma, beta, residual=residual)
    routing = ep.route_topk(logits, 8, scoring="sigmoid", groups=8, topk_groups=4)
    balance = ep.balance_loss(logits, routing.ids, scoring="sigmoid", sequence_offsets=offsets)
    from_balance = ep.balance_loss_backward(torch.ones_like(balance.loss), logits, routing.ids, balance.counts, balance.tokens, scoring="sigmoid",
                                            sequence_offsets=offsets)
    from_weights = ep.route_topk_backward(grad_weights, logits, routing.ids, scoring="sigmoid")
    grads = ep.layer_norm_backward(grad, normed.residual, gamma, normed.mean, normed.rstd, grad_residual=grad)
    return normed.normalized, normed.residual, routing.ids, routing.weights, balance.loss, balance.counts, from_balance, from_weights, *grads


def make_entry(device, seed, tokens=700, hidden=1024, experts=64):
    x, residual, gamma, beta = make_norm(tokens, hidden, BF16, BF16, seed)
    return [*to(device, x, residual, gamma, beta, 2 * randn(seed + 4, tokens, experts), randn(seed + 5, tokens, hidden).to(BF16), randn(seed + 6, tokens, 8)),
            torch.tensor([0, 100, 430, 690], device=device)]


def test_captured_entries_replay(device):
    """Two graphs of the same calls, replayed in turn with new inputs and eager calls between them."""
    states, graphs = [make_entry(device, seed) for seed in (101, 111)], []
    for state in states:
        for _ in range(2):
            entry(*state)
    torch.cuda.synchronize()
    for state in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = entry(*state)
        graphs.append((graph, outputs))
    for turn in range(4):
        print("replay", turn, flush=True)
        fresh = [make_entry(device, 200 + 10 * turn + i) for i in range(2)]
        for state, new in zip(states, fresh):
            for tensor, value in zip(state[:-1], new[:-1]):
                tensor.copy_(value)
        for graph, _ in graphs:
            graph.replay()
        want = [entry(*new) for new in fresh]
        torch.cuda.synchronize()
        for (_, outputs), values in zip(graphs, want):
            for got, value in zip(outputs, values):
                assert same_bits(got, value)


def test_a_captured_step_with_its_gradients_replays(device):
    """Autograd's own passes in a graph: captured when no eager result of the same leaves is left."""
    x, residual, gamma, beta, logits, grad, grad_weights, offsets = make_entry(device, 121)
    share = torch.tensor([0.5, 1.0, 2.0], device=device)

    def step(*leaves):
        x, residual, gamma, beta, logits = leaves
        entered = ep.layer_norm(x, gamma, beta, residual=residual)
        routing = ep.route_topk(logits, 8, scoring="sigmoid")
        balance = ep.balance_loss(logits, routing.ids, scoring="sigmoid", sequence_offsets=offsets)
        found = torch.autograd.grad((entered.normalized, entered.residual, routing.weights, balance.loss), leaves, (grad, grad, grad_weights, share))
        return [*found, entered.normalized.detach(), routing.weights.detach(), balance.loss.detach()]

    leaves = [tensor.clone().requires_grad_() for tensor in (x, residual, gamma, beta, logits)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step(*leaves)
    for turn in range(4):
        print("replay of a step", turn, flush=True)
        fresh = make_entry(device, 300 + 10 * turn)
        with torch.no_grad():
            for leaf, value in zip(leaves, fresh):
                leaf.copy_(value)
        graph.replay()
        want = step(*(value.requires_grad_() for value in fresh[:5]))
        torch.cuda.synchronize()
        for got, value in zip(outputs, want):
            assert same_bits(got, value)


def test_entries_at_once_on_two_streams(device):
    states = [make_entry(device, seed) for seed in (121, 131)]
    want = [entry(*state) for state in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(5):
        results = []
        for state, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                results.append(entry(*state))
        torch.cuda.synchronize()
        for got, values in zip(results, want):
            assert all(same_bits(a, b) for a, b in zip(got, values))


def test_a_layer_is_trained_from_its_entry_to_its_output(device):
    """Norm, router, dispatch, experts, combine and the balance loss, forward and backward through autograd, against the same in fp32
    elementary operations with the choices given."""
    tokens, hidden, experts, topk, weight = 257, 512, 12, 3, 0.1
    x, residual, gamma, _ = make_norm(tokens, hidden, BF16, FP32, 141)
    gains, router, grad = 1 + 0.1 * randn(142, experts, hidden), randn(143, experts, hidden) / hidden**0.5, randn(144, tokens, hidden).to(BF16)
    x, residual, gamma, gains, router, grad = to(device, x, residual, gamma, gains.to(BF16), router, grad)
    leaves = [tensor.requires_grad_() for tensor in (x, residual, gamma, gains, router)]
    with ep.Buffer(None, ep.EPConfig(experts, topk, hidden, tokens)) as buffer:
        normed = ep.rms_norm(x, gamma, residual=residual)
        logits = normed.normalized.float() @ router.T
        routing = ep.route_topk(logits, topk)
        handle = buffer.dispatch(normed.normalized.detach(), topk_idx=routing.ids, do_expand=True, alignment=16).handle
        layout = handle.layout
        rows = ep.dispatch_rows(buffer, normed.normalized, handle)
        slot = torch.arange(rows.shape[0], device=device)
        expert = torch.searchsorted(layout.expert_offsets[1:].contiguous(), slot, right=True).clamp(max=experts - 1)
        out = ep.combine_weighted(rows * gains[expert], handle.token_slots, routing.weights, bias=normed.residual,
                                  expert_offsets=layout.expert_offsets, expert_counts=layout.expert_counts)
        balance = ep.balance_loss(logits, routing.ids)
        assert torch.equal(balance.counts, layout.expert_counts)
        loss = (out.float() * grad.float()).sum() + weight * balance.loss
        found = torch.autograd.grad(loss, leaves)
    ids = routing.ids
    s = x.float() + residual.float()
    n = s * (s.square().mean(1, keepdim=True) + 1e-6).rsqrt() * gamma
    wide = n @ router.T
    w = torch.softmax(wide.gather(1, ids), dim=1)
    dense = s + (n[:, None] * gains.float()[ids] * w[:, :, None]).sum(1)
    even = experts * (balance.counts / balance.counts.sum() * torch.softmax(wide, dim=1).mean(0)).sum()
    want = torch.autograd.grad((dense * grad.float()).sum() + weight * even, leaves)
    # bf16 activations and gradients: a handful of roundings of 2^-8 each
    for got, value in zip((out, *found), (dense, *want)):
        assert (got.float() - value.float()).norm() <= 2.0**-5 * value.float().norm()


# ------------------------------------------------------------------ refusals


def test_entry_refusals(device):
    x, residual, gamma, beta = to(device, *make_norm(4, 256, BF16, BF16, 151))
    logits, ids = torch.randn(4, 16, device=device), torch.zeros(4, 2, dtype=torch.int64, device=device)
    weights, stat = torch.ones(4, 2, device=device), torch.ones(4, device=device)
    offsets = torch.tensor([0, 4], device=device)
    counts, tokens = torch.ones(16, dtype=torch.int64, device=device), torch.ones((), dtype=torch.int64, device=device)
    half, odd = x.half(), torch.zeros(4, 252, dtype=BF16, device=device)
    off = torch.zeros(4 * 256 + 1, dtype=BF16, device=device)[1:].view(4, 256)
    calls = [
        lambda: ep.layer_norm(half, half[0]), lambda: ep.layer_norm(odd, odd[0]), lambda: ep.layer_norm(x[0], gamma), lambda: ep.layer_norm(x.T, gamma),
        lambda: ep.layer_norm(off, gamma), lambda: ep.layer_norm(x, gamma[:8]), lambda: ep.layer_norm(x, gamma, beta.float()),
        lambda: ep.layer_norm(x, gamma.half()), lambda: ep.layer_norm(x.float(), gamma), lambda: ep.layer_norm(x, gamma, residual=residual.float()),
        lambda: ep.layer_norm(x, gamma, residual=residual[:3]), lambda: ep.layer_norm(x, gamma, residual=off), lambda: ep.layer_norm(x, gamma, eps=-1.0),
        lambda: ep.rms_norm(x, gamma, eps=math.nan), lambda: ep.rms_norm(x, gamma.cpu()), lambda: ep.rms_norm(torch.zeros(1, 16392, dtype=BF16, device=device), gamma),
        lambda: ep.layer_norm_backward(x.float(), x, gamma, stat, stat), lambda: ep.layer_norm_backward(x, x, gamma, stat[:3], stat),
        lambda: ep.layer_norm_backward(x, x, gamma, stat, stat.double()), lambda: ep.layer_norm_backward(x[:3], x, gamma, stat, stat),
        lambda: ep.rms_norm_backward(x, x, gamma, stat, grad_residual=x[:2]), lambda: ep.rms_norm_backward(off, x, gamma, stat),
        lambda: ep.rms_norm_backward(x, x, gamma, stat, input=False, parameters=False),
        lambda: ep.route_topk(logits.half(), 2), lambda: ep.route_topk(logits[0], 2), lambda: ep.route_topk(logits, 0), lambda: ep.route_topk(logits, 17),
        lambda: ep.route_topk(torch.zeros(1, 4097, device=device), 2), lambda: ep.route_topk(torch.zeros(1, 64, device=device), 33),
        lambda: ep.route_topk(logits.T, 2), lambda: ep.route_topk(logits[:1].expand(4, 16), 2), lambda: ep.route_topk(logits, 2, scoring="tanh"),
        lambda: ep.route_topk(logits, 2, bias=torch.zeros(15, device=device)), lambda: ep.route_topk(logits, 2, bias=torch.zeros(16, dtype=BF16, device=device)),
        lambda: ep.route_topk(logits, 2, bias=torch.zeros(16)), lambda: ep.route_topk(logits, 2, mask=torch.ones(4, device=device)),
        lambda: ep.route_topk(logits, 2, mask=torch.ones(3, dtype=torch.bool, device=device)), lambda: ep.route_topk(logits, 2, groups=3),
        lambda: ep.route_topk(logits, 2, groups=0), lambda: ep.route_topk(logits, 2, groups=4, topk_groups=5), lambda: ep.route_topk(logits, 8, groups=4, topk_groups=1),
        lambda: ep.route_topk(torch.zeros(1, 130, device=device), 2, groups=65, topk_groups=2),
        lambda: ep.route_topk_backward(weights, logits, ids.int()), lambda: ep.route_topk_backward(weights[:, :1], logits, ids),
        lambda: ep.route_topk_backward(weights.double(), logits, ids), lambda: ep.route_topk_backward(weights, logits, ids[:3]),
        lambda: ep.route_topk_backward(torch.ones(4, 33, device=device), logits, torch.zeros(4, 33, dtype=torch.int64, device=device)),
        lambda: ep.balance_loss(logits, ids.int()), lambda: ep.balance_loss(logits, ids[:3]), lambda: ep.balance_loss(logits, ids, scoring="none"),
        lambda: ep.balance_loss(logits, ids, sequence_offsets=offsets[:1]), lambda: ep.balance_loss(logits, ids, sequence_offsets=offsets.int()),
        lambda: ep.balance_loss(logits, ids, sequence_offsets=offsets.cpu()), lambda: ep.balance_loss(logits, ids, sequence_offsets=offsets.view(1, 2)),
        lambda: ep.balance_loss_backward(weights, logits, ids, counts, tokens), lambda: ep.balance_loss_backward(tokens.float(), logits, ids, counts[:8], tokens),
        lambda: ep.balance_loss_backward(tokens.float(), logits, ids, counts, tokens, sequence_offsets=offsets),
    ]
    for number, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {number} was taken")


def test_derivatives_that_do_not_exist_are_refused(device):
    from torch.autograd import forward_ad

    x, _, gamma, beta = to(device, *make_norm(4, 256, FP32, FP32, 153))
    logits, ids = torch.randn(4, 16, device=device), torch.zeros(4, 2, dtype=torch.int64, device=device)
    weights, stat = torch.ones(4, 2, device=device), torch.ones(4, device=device)
    counts, tokens, loss = torch.ones(16, dtype=torch.int64, device=device), torch.ones((), dtype=torch.int64, device=device), torch.ones((), device=device)
    calls = [(lambda x: ep.layer_norm(x, gamma, beta), x), (lambda g: ep.layer_norm(x, g, beta), gamma), (lambda x: ep.rms_norm(x, gamma), x),
             (lambda x: ep.rms_norm(gamma.new_zeros(4, 256), gamma, residual=x), x),
             (lambda logits: ep.route_topk(logits, 2), logits), (lambda logits: ep.balance_loss(logits, ids), logits),
             (lambda x: ep.layer_norm_backward(x, x.detach(), gamma, stat, stat), x), (lambda x: ep.rms_norm_backward(x, x.detach(), gamma, stat), x),
             (lambda w: ep.route_topk_backward(w, logits, ids), weights), (lambda g: ep.balance_loss_backward(g, logits, ids, counts, tokens), loss)]
    for number, (call, value) in enumerate(calls):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(value, torch.ones_like(value))
            with pytest.raises(RuntimeError):
                call(dual)
                pytest.fail(f"call {number} dropped a forward-mode derivative")
    for call, value in calls[6:]:
        with pytest.raises(RuntimeError, match="has no gradient"):
            call(value.clone().requires_grad_())
    for call, value, out in ((lambda x: ep.layer_norm(x, gamma, beta).normalized, x, None), (lambda v: ep.route_topk(v, 2).weights, logits, None),
                             (lambda v: ep.balance_loss(v, ids).loss, logits, None)):
        leaf = value.clone().requires_grad_()
        (first,) = torch.autograd.grad(call(leaf).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.sum(), leaf)
