"""The router and the balance loss at extreme logits, and groups of scores that are tiny, lost, infinite or NaN, where fp32 has nothing left
to tell values apart by.

Choices go by values in 64 bits, found here one by one (a library's vectorised sigmoid may give equal logits two values).  Inputs are such that
values which are not equal differ by far more than a last bit of 64."""

import math

import pytest
import torch

import entry_oracle as oracle
import nanoep_amd as ep
from test_gpu_entry import BF16, FP32, SCORINGS, check_balance, check_route, make_balance, randn, same_bits

pytestmark = pytest.mark.gpu


def values_of(logits, scoring, bias):
    """A token's scores plus bias: a softmax's numerators where there is none, since their sum is a factor of all."""
    top = max((v for v in logits if v == v), default=0.0)
    top = 0.0 if top == -math.inf else top

    def exp(v):
        return v if v != v else math.inf if v > 709.0 else math.exp(v)

    if scoring == "sigmoid":
        values = [1.0 / (1.0 + exp(-v)) for v in logits]
    else:
        values = [exp(v - top) for v in logits]
        if bias is not None:
            total = sum(values) or 1.0  # (nothing but -infinity: nothing is left in any case)
            values = [v / total for v in values]
    return values if bias is None else [v + b for v, b in zip(values, bias)]


def descending(value):
    return (0, 0.0) if value != value else (1, -value)  # NaN ahead of everything


def choose_of_token(logits, topk, scoring, bias, groups, topk_groups):
    values = values_of(logits, scoring, bias)
    left = [e for e, v in enumerate(values) if logits[e] != -math.inf and v != -math.inf]
    size = len(logits) // groups
    of_group = []
    for g in range(groups):
        best = sorted((values[e] for e in left if e // size == g), key=descending)[:2]
        if best:
            of_group.append((sum(best), g))
    kept = {g for _, g in sorted(of_group, key=lambda entry: (descending(entry[0]), entry[1]))[:topk_groups]}
    chosen = sorted((e for e in left if e // size in kept), key=lambda e: (descending(values[e]), e))[:topk]
    return chosen + [-1] * (topk - len(chosen))


def choose(logits, topk, scoring, bias, groups, topk_groups):
    bias = None if bias is None else bias.double().tolist()
    return torch.tensor([choose_of_token(row, topk, scoring, bias, groups, topk_groups) for row in logits.double().tolist()])


def route(device, logits, topk, bias, **options):
    return ep.route_topk(logits.to(device), topk, bias=None if bias is None else bias.to(device), **options)


def check_groups(device, logits, topk, scoring, bias, groups, topk_groups, normalize=True):
    """A batch, and each of its tokens as a call of its own: the ids of the definition, and the batch's bits."""
    options = {"scoring": scoring, "groups": groups, "topk_groups": topk_groups, "normalize": normalize}
    got = route(device, logits, topk, bias, **options)
    want = choose(logits, topk, scoring, bias, groups, topk_groups)
    wrong = (got.ids.cpu() != want).any(1).nonzero().flatten().tolist()
    assert not wrong, [(t, got.ids[t].tolist(), want[t].tolist()) for t in wrong[:4]]
    for t in range(min(logits.shape[0], 24)):
        one = route(device, logits[t : t + 1], topk, bias, **options)
        assert same_bits(one.ids[0], got.ids[t]) and same_bits(one.weights[0], got.weights[t]), t
    return got


def extreme(experts, dtype, seed):
    lowest = torch.finfo(dtype).min
    logits = randn(seed, 16, experts)
    logits[1] = -88.0  # sigmoids at the end of fp32's range, and beyond it
    logits[2] = -89.0
    logits[3] = -120.0
    logits[4] = lowest  # masked with the type's lowest value: experts like others
    logits[5, 3:] = lowest
    logits[6, : experts // 2] = lowest
    logits[7] -= 90.0
    logits[8] = -200.0 - torch.arange(experts)
    logits[9] = 80.0 + torch.arange(experts) % 32
    logits[10] = -math.inf
    logits[11, 1:] = -math.inf
    logits[12] = -95.0
    logits[12, experts // 2 :] = -math.inf
    logits[13] *= 30.0
    logits[14, 5] = 1e30  # all other numerators are zero
    return logits.to(dtype)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("experts,groups,topk_groups,topk", [(16, 16, 5, 4), (64, 8, 3, 6), (60, 3, 2, 6), (256, 4, 2, 8), (256, 64, 40, 8)])
def test_groups_of_extreme_logits(device, scoring, biased, dtype, experts, groups, topk_groups, topk):
    print("groups, extreme", scoring, biased, dtype, experts, groups, flush=True)
    bias = 0.01 * randn(102, experts) if biased else None
    check_groups(device, extreme(experts, dtype, 101), topk, scoring, bias, groups, topk_groups)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("experts,groups,topk_groups,topk", [(64, 8, 3, 6), (60, 3, 2, 6), (256, 4, 2, 8)])
def test_groups_of_nan_and_infinity(device, scoring, biased, experts, groups, topk_groups, topk):
    logits = randn(103, 8, experts)
    logits[1, 17] = math.inf
    logits[2, 17] = math.nan
    logits[3] = math.nan
    logits[4, [3, experts - 1]] = math.inf
    logits[5, [3, experts - 1]] = math.nan
    logits[6, 17], logits[6, 0] = math.inf, math.nan
    bias = 0.01 * randn(104, experts) if biased else None
    print("groups, nan", scoring, biased, experts, groups, flush=True)
    got = check_groups(device, logits, topk, scoring, bias, groups, topk_groups)
    assert got.weights[[0, 7]].isfinite().all()


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_groups_of_sigmoids_that_end_within_fp32s_range(device, dtype):
    """Two sigmoids that fp32 loses against one that it holds: at e^-88.7 their exponential overflows, from e^-87.3 on results lose digits."""
    experts, groups = 16, 2
    logits = torch.full((12, experts), -200.0)
    for t, (two, one) in enumerate([(-89.0, -88.5), (-87.5, -87.0), (-88.75, -88.25), (-88.0, -87.5), (-90.0, -89.5), (-87.25, -86.75)]):
        for group in (0, 1):  # the two are worth more, wherever they are
            logits[2 * t + group, [8 * group + 2, 8 * group + 5]] = two
            logits[2 * t + group, 8 * (1 - group) + 3] = one
    print("groups, end of the range", dtype, flush=True)
    check_groups(device, logits.to(dtype), 2, "sigmoid", None, groups, 1)
    check_groups(device, (-86.0 - 4.0 * torch.rand(200, 64, generator=torch.Generator().manual_seed(105))).to(dtype), 6, "sigmoid", None, 8, 3)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("experts,topk", [(32, 8), (256, 8), (256, 1)])
def test_experts_whose_scores_end_within_fp32s_range(device, scoring, experts, topk):
    """Candidates of a group whose numerators or sigmoids have few digits left, or none."""
    generator = torch.Generator().manual_seed(106)
    logits = -84.0 - 22.0 * torch.rand(200, experts, generator=generator)
    if scoring == "softmax":
        logits[:, 0] = 0.0
        logits[100:] += 40.0  # differences are rounded
    logits[::2, 1:] = logits[::2, 1:].clamp(max=-95.0)
    print("experts, end of the range", scoring, experts, topk, flush=True)
    check_groups(device, logits, topk, scoring, None, 2, 1)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("groups,biased", [(1, False), (1, True), (4, False), (4, True)])
def test_weights_of_tokens_with_nan_or_infinity(device, scoring, normalize, groups, biased):
    """All of a token's weights, but of plain sigmoids the NaN's own alone; an infinity breaks a softmax and no sigmoid."""
    experts, topk = 64, 6
    logits = randn(107, 5, experts)
    logits[1, [17, 40]] = math.nan
    logits[2, 17] = math.inf
    logits[3, 17], logits[3, 40] = math.inf, math.nan
    bias = 0.01 * randn(108, experts) if biased else None
    print("weights, nan", scoring, normalize, groups, biased, flush=True)
    got = route(device, logits, topk, bias, scoring=scoring, normalize=normalize, groups=groups, topk_groups=max(1, groups // 2))
    ids, broken = got.ids.cpu(), got.weights.cpu().isnan()
    expected = torch.zeros(5, topk, dtype=torch.bool)
    if scoring == "softmax":
        expected[1:4] = True
    elif normalize:
        expected[[1, 3]] = True
    else:
        expected = logits.gather(1, ids).isnan()
        assert expected.sum(1).tolist() == [0, 2, 0, 1, 0]
    assert torch.equal(broken, expected)
    fine = ~broken.any(1)
    weights, slack = oracle.weigh(logits[fine], ids[fine], scoring, normalize, 1.0)
    assert ((got.weights.cpu()[fine] - weights).abs() <= slack).all()


@pytest.fixture
def tight(monkeypatch):
    """The oracle's bounds for logits of any size.  What is rounded is the difference of a logit and its token's largest, by 2^-24 of itself,
    however large the two are; and e^-110 (the largest being e^0) is zero to within LEAST, so no difference above that rounds anything."""

    def spread(logits):
        logits, finite = logits.double(), logits.isfinite()
        top = logits.masked_fill(~finite, -math.inf).amax(1, keepdim=True)
        return (top - logits.masked_fill(~finite, math.inf).amin(1, keepdim=True)).clamp(min=0.0, max=110.0)

    monkeypatch.setattr(oracle, "_spread", spread)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("experts,topk", [(16, 3), (60, 6), (256, 8)])
def test_weights_and_gradients_of_extreme_logits(device, tight, scoring, normalize, dtype, experts, topk):
    logits, grad = extreme(experts, dtype, 109), randn(110, 16, topk)
    print("weights, extreme", scoring, normalize, dtype, experts, flush=True)
    got = check_route(device, logits, topk, scoring=scoring, normalize=normalize)
    some = [t for t in range(16) if t != 10]  # (the one has no softmax)
    # the router's own choices, and others, some of experts that could not have been chosen
    for ids in (got.ids.cpu()[some], torch.randint(-1, experts, (len(some), topk), generator=torch.Generator().manual_seed(111))):
        found = ep.route_topk_backward(grad[some].to(device), logits[some].to(device), ids.to(device), scoring=scoring, normalize=normalize)
        oracle.check_rounded(found, *oracle.weigh_backward(grad[some], logits[some], ids, scoring, normalize, 1.0), dtype)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("experts,topk", [(16, 3), (60, 6), (256, 8)])
@pytest.mark.parametrize("offsets", [None, [0, 5, 5, 30, 48]])
def test_balance_loss_of_extreme_logits(device, tight, scoring, dtype, experts, topk, offsets):
    logits, ids = make_balance(48, experts, topk, 112, dtype)
    logits[::3] = extreme(experts, dtype, 113)
    print("balance, extreme", scoring, dtype, experts, offsets, flush=True)
    got, grad = check_balance(device, logits, ids, scoring, offsets)
    assert got.loss.isfinite().all() and grad.isfinite().all()


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("experts,topk", [(7, 2), (16, 8), (32, 8), (60, 6), (64, 16), (100, 8), (200, 4), (256, 8), (400, 16), (512, 2)])
def test_a_tokens_choice_is_the_same_bits_in_any_batch(device, scoring, experts, topk):
    """Batches of fewer and of more tokens than a device has 32 lanes for."""
    logits = (2 * randn(114, 9001, experts)).to(device)
    bias = (0.1 * randn(115, experts)).to(device)
    print("same bits in any batch", scoring, experts, topk, flush=True)
    for normalize in (True, False):
        for options in ({}, {"bias": bias}):
            whole = ep.route_topk(logits, topk, scoring=scoring, normalize=normalize, **options)
            for first, last in ((0, 1), (9000, 9001), (1000, 3047)):
                part = ep.route_topk(logits[first:last], topk, scoring=scoring, normalize=normalize, **options)
                assert same_bits(part.ids, whole.ids[first:last]) and same_bits(part.weights, whole.weights[first:last]), (normalize, list(options), first)


@pytest.mark.parametrize("offsets", [None, [0, 100, 260]])
def test_counts_may_be_reduced_ahead_of_the_backward_pass(device, offsets):
    """In place, as a collective over ranks does it, which autograd does not see (as it does not see changes of `data`)."""
    logits, ids = make_balance(300, 60, 6, 116)
    logits, ids = logits.to(device).requires_grad_(), ids.to(device)
    bounds = None if offsets is None else torch.tensor(offsets, device=device)
    print("counts, reduced", offsets, flush=True)

    def found(change):
        balance = ep.balance_loss(logits, ids, sequence_offsets=bounds)
        change(balance)
        return torch.autograd.grad(balance.loss.sum(), logits)[0]

    def unseen(balance):
        balance.counts.data.add_(torch.arange(60, device=device))
        balance.tokens.data.mul_(2)

    def seen(balance):
        balance.counts.mul_(3)
        balance.tokens.zero_()

    want = found(lambda balance: None)
    assert same_bits(found(unseen), want) and same_bits(found(seen), want)


@pytest.mark.parametrize("experts", [1, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 512, 513, 1024, 1025, 2048, 2049, 4096])
def test_every_spread_of_experts_over_lanes(device, experts):
    """Both sides of every size at which a token takes more lanes or a lane more experts, in short and in long batches.

    Bounds, relative to sums of positive terms: a sigmoid's derivative has two exponentials and six roundings, 20 * 2^-22 with the topk
    additions' shares; shares are off by 2 (20 * 2^-24 + 2^-22) + 104 * 2^-24 < 1e-5, the losses' products of up to three such by less than 1e-4."""
    logits = randn(117, 8300, experts).to(device)
    for topk in (1, 8, 9, 16, 17, 32):
        print("spreads", experts, topk, flush=True)
        for tokens in (3, 8300):
            part, some = logits[:tokens], min(topk, experts)
            want = part.sort(dim=1, descending=True, stable=True).indices[:, :some]
            got = ep.route_topk(part, some)
            assert torch.equal(got.ids, want)
            assert torch.equal(ep.route_topk(part, some, scoring="sigmoid", bias=torch.zeros(experts, device=device)).ids, want)
            for groups in (2, 33, 64):
                if experts % groups == 0 and some <= experts - experts // groups:
                    within = ep.route_topk(part, some, scoring="sigmoid", groups=groups, topk_groups=groups - 1).ids
                    assert torch.equal(within[:3].cpu(), choose(part[:3].cpu(), some, "sigmoid", None, groups, groups - 1))
            ids = torch.randint(0, experts, (tokens, topk), device=device, generator=torch.Generator(device).manual_seed(118))
            grad = ep.route_topk_backward(torch.ones(tokens, topk, device=device), part, ids, scoring="sigmoid", normalize=False)
            sigmoids = torch.sigmoid(part.double())
            want = torch.zeros_like(sigmoids).scatter_add_(1, ids, torch.ones(tokens, topk, device=device, dtype=torch.float64)) * sigmoids * (1 - sigmoids)
            assert ((grad - want).abs() <= topk * 20 * oracle.EXP * want + oracle.LEAST).all()
            balance = ep.balance_loss(part, ids)
            assert torch.equal(balance.counts, torch.bincount(ids.view(-1), minlength=experts)) and int(balance.tokens) == tokens
            loss_grad = ep.balance_loss_backward(torch.ones((), device=device), part, ids, balance.counts, balance.tokens)
            p = torch.softmax(part.double(), dim=1)
            f = experts * balance.counts.double() / (tokens * topk) / tokens
            want = p * (f - (p * f).sum(1, keepdim=True))
            assert ((loss_grad - want).abs() <= 1e-4 * p * f.max() + oracle.LEAST).all()
            assert abs(float(balance.loss) - float((f * p).sum())) <= 1e-4 * float(balance.loss)
