"""The expert layer's operators on the GPU against their definitions in 64 bits."""

import pytest
import torch

import nanoep_amd as ep
import operator_oracle as oracle

pytestmark = pytest.mark.gpu

NAN_BYTE = 0x7F


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def close(got, want, slack):
    """bf16 results: the correct rounding of some value within `slack` of the exact one."""
    assert got.shape == want.shape and got.dtype == torch.bfloat16
    low, high = (want - slack).to(torch.bfloat16), (want + slack).to(torch.bfloat16)
    got = got.cpu()
    assert ((low <= got) & (got <= high)).all()


# ------------------------------------------------------------------ norm


@pytest.mark.parametrize("hidden", [16, 112, 128, 240, 1024, 2816, 7168, 8208, 65536])
@pytest.mark.parametrize("tokens", [1, 3, 1025])
@pytest.mark.parametrize("options", ["plain", "residual", "both"])
def test_rms_norm(device, tokens, hidden, options):
    if tokens > 3 and hidden > 8208:
        tokens = 33
    x = (3 * randn(hidden, tokens, hidden)).to(torch.bfloat16)
    residual = randn(tokens, tokens, hidden).to(torch.bfloat16) if options != "plain" else None
    gamma = (1 + 0.2 * randn(5, hidden)).to(torch.bfloat16)
    print("rms_norm_fp8", tokens, hidden, options, flush=True)
    got = ep.rms_norm_fp8(x.to(device), gamma.to(device), residual=None if residual is None else residual.to(device), eps=1e-5,
                          normalized=options == "both")
    s, n, slack = oracle.rms_norm(x, residual, gamma, 1e-5)
    oracle.check_eight_bits(got.rows.values.cpu(), got.rows.scales.cpu(), n, slack)
    assert (got.residual is None) == (residual is None) and (got.normalized is None) == (options != "both")
    if residual is not None:
        close(got.residual, s, s.abs() * oracle.FP32)
    if options == "both":
        close(got.normalized, n, slack)
    # the record behind the two views: what they hold, and zeros
    width = ep.fp8_payload_width(hidden)
    assert got.rows.payload.shape == (tokens, width)
    again = ep.Fp8Rows.of_payload(got.rows.payload, hidden)
    assert torch.equal(again.values.view(torch.uint8), got.rows.values.view(torch.uint8)) and torch.equal(again.scales, got.rows.scales)
    used = hidden + 4 * oracle.groups(hidden)
    assert not got.rows.payload.view(torch.uint8)[:, used:].any()


def test_rms_norm_of_zeros_infinities_and_nan(device):
    x = randn(1, 5, 512).to(torch.bfloat16)
    x[0] = 0
    x[1, 128:256] = 0
    x[2, 300] = float("inf")
    x[3, 300] = float("nan")
    gamma = torch.ones(512, dtype=torch.bfloat16)
    got = ep.rms_norm_fp8(x.to(device), gamma.to(device), eps=0.0, normalized=True)
    values, scales = got.rows.values.cpu().float(), got.rows.scales.cpu()
    # 0 / 0 without an eps; zeros in a group of an ordinary row stay zeros under the smallest scale
    assert values[0].isnan().all() and scales[0].isnan().all()
    assert not values[1, 128:256].any() and (scales[1, 1] == oracle.SMALLEST_AMAX / oracle.LARGEST).all()
    # an infinity: the row's factor is 0, its own place 0 * inf
    assert not values[2, :256].any() and scales[2, 2].isnan() and values[2, 300].isnan()
    assert values[3].isnan().all() and scales[3].isnan().all()
    assert values[4].isfinite().all() and scales[4].isfinite().all() and got.normalized.cpu()[4].isfinite().all()
    zeros = ep.rms_norm_fp8(torch.zeros(2, 512, dtype=torch.bfloat16, device=device), gamma.to(device))
    assert not zeros.rows.values.float().any() and (zeros.rows.scales == oracle.SMALLEST_AMAX / oracle.LARGEST).all()


def test_rms_norm_of_no_tokens(device):
    empty = torch.empty(0, 256, dtype=torch.bfloat16, device=device)
    got = ep.rms_norm_fp8(empty, torch.ones(256, dtype=torch.bfloat16, device=device), residual=empty, normalized=True)
    assert got.rows.values.shape == (0, 256) and got.rows.scales.shape == (0, 2) and got.residual.shape == got.normalized.shape == (0, 256)


# ------------------------------------------------------------------ products

# counts of the experts and the alignment of their segments; rows behind the last one
SEGMENTS = {
    "single row": ([1], 1, 0),
    "one expert": ([37], 1, 0),
    "small": ([0, 1, 5, 0, 16, 17, 2], 1, 0),
    "padded": ([3, 0, 16, 33, 1], 16, 0),
    "long gap": ([1, 0, 130], 128, 40),
    "uneven": ([200, 3, 0, 65, 300], 1, 7),
    "many": ([(7 * e) % 5 for e in range(150)], 1, 0),
    "none": ([0, 0, 0], 1, 9),
    "large": ([500, 260, 129, 0, 255], 128, 0),
}
SIZES = [(16, 32), (128, 256), (144, 96), (256, 288), (1424, 512), (640, 1056)]


def make_product(segments, inner, columns, seed, gap_byte=NAN_BYTE):
    counts, alignment, behind = SEGMENTS[segments]
    counts = torch.tensor(counts)
    padded = (counts + alignment - 1) // alignment * alignment
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), padded.cumsum(0)])
    rows = int(offsets[-1]) + behind
    values, scales = oracle.quantize_rows(randn(seed, rows, inner) * (1 + randn(seed + 1, rows, 1).abs()))
    # nobody looks at rows of no expert
    owned = torch.zeros(rows, dtype=torch.bool)
    for e in range(len(counts)):
        owned[offsets[e] : offsets[e] + counts[e]] = True
    values.view(torch.uint8)[~owned] = gap_byte
    scales[~owned] = float("nan")
    weight = ep.quantize_weight(randn(seed + 2, len(counts), columns, inner) / inner**0.5)
    return values, scales, weight, offsets, counts


def records_of(values, scales, device):
    """The rows as a dispatch hands them out: views of records."""
    rows, inner = values.shape
    payload = torch.full((rows, ep.fp8_payload_width(inner)), float("nan"), dtype=torch.bfloat16)
    view = ep.Fp8Rows.of_payload(payload, inner)
    view.values.view(torch.uint8).copy_(values.view(torch.uint8))
    view.scales.copy_(scales)
    return ep.Fp8Rows.of_payload(payload.to(device), inner)


def on(device, weight):
    return ep.Fp8Weight(weight.values.to(device), weight.scales.to(device))


# the kernel by the product's size, and each one whatever its size
KERNELS = [0, 1, 64, 128, 256]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("inner,columns", SIZES)
@pytest.mark.parametrize("segments", SEGMENTS)
def test_experts_linear(device, tuning, segments, inner, columns, kernel):
    tuning("EXPERTS_TILE", kernel)
    columns -= 8 if inner == 144 else 0  # a tile of columns that ends early
    values, scales, weight, offsets, counts = make_product(segments, inner, columns, inner + columns)
    z, slack = oracle.experts(values, scales, weight.values, weight.scales, offsets, counts)
    print("experts_linear", segments, inner, columns, kernel, flush=True)
    got = ep.experts_linear(records_of(values, scales, device), on(device, weight), offsets.to(device), counts.to(device))
    close(got, z, slack)
    loose = ep.Fp8Rows(values.to(device), scales.to(device))
    assert torch.equal(ep.experts_linear(loose, on(device, weight), offsets.to(device), counts.to(device)), got)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("inner,columns", SIZES)
@pytest.mark.parametrize("segments", SEGMENTS)
def test_experts_gated(device, tuning, segments, inner, columns, kernel):
    tuning("EXPERTS_TILE", kernel)
    values, scales, weight, offsets, counts = make_product(segments, inner, columns, inner + columns)
    act, slack = oracle.gated(*oracle.experts(values, scales, weight.values, weight.scales, offsets, counts))
    print("experts_gated", segments, inner, columns, kernel, flush=True)
    got = ep.experts_gated(records_of(values, scales, device), on(device, weight), offsets.to(device), counts.to(device))
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), act, slack)
    width = columns // 2
    assert not got.payload.view(torch.uint8)[:, width + 4 * oracle.groups(width) :].any()
    again = ep.experts_gated(records_of(values, scales, device), on(device, weight), offsets.to(device), counts.to(device))
    assert torch.equal(again.payload.view(torch.int16), got.payload.view(torch.int16))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("alignment", [1, 16])
def test_products_of_counts_around_every_row_tile(device, tuning, monkeypatch, alignment, kernel):
    """A matrix instruction has 16 rows; tiles leave out those of their row tiles that hold no row."""
    tuning("EXPERTS_TILE", kernel)
    counts = [16 * tiles + more for tiles in range(9) for more in (-1, 0, 1) if 16 * tiles + more > 0]
    monkeypatch.setitem(SEGMENTS, "edges", (counts, alignment, 5))
    values, scales, weight, offsets, counts = make_product("edges", 272, 288, 31 + alignment)
    z, slack = oracle.experts(values, scales, weight.values, weight.scales, offsets, counts)
    rows, weight, layout = records_of(values, scales, device), on(device, weight), (offsets.to(device), counts.to(device))
    print("counts around row tiles", alignment, kernel, flush=True)
    close(ep.experts_linear(rows, weight, *layout), z, slack)
    got = ep.experts_gated(rows, weight, *layout)
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), *oracle.gated(z, slack))


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("kernel", KERNELS)
def test_products_without_a_layout_are_one_experts(device, rows, tuning, kernel):
    tuning("EXPERTS_TILE", kernel)
    inner, columns = 272, 320
    values, scales = oracle.quantize_rows(randn(rows, rows, inner))
    weight = ep.quantize_weight(randn(rows + 1, 1, columns, inner))
    z, slack = oracle.experts(values, scales, weight.values, weight.scales, None, None)
    rows_on = ep.Fp8Rows(values.to(device), scales.to(device))
    print("products without a layout", rows, flush=True)
    close(ep.experts_linear(rows_on, on(device, weight)), z, slack)
    got = ep.experts_gated(rows_on, on(device, weight))
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), *oracle.gated(z, slack))


@pytest.mark.parametrize("kernel", KERNELS)
def test_products_follow_strides_of_their_own(device, tuning, kernel):
    tuning("EXPERTS_TILE", kernel)
    values, scales, weight, offsets, counts = make_product("uneven", 256, 128, 9)
    z, slack = oracle.experts(values, scales, weight.values, weight.scales, offsets, counts)
    rows = values.shape[0]
    wide = torch.full((rows, 256 + 48), NAN_BYTE, dtype=torch.uint8, device=device)
    wide[:, :256] = values.view(torch.uint8).to(device)
    wide_scales = torch.full((rows, 5), float("nan"), device=device)
    wide_scales[:, 2:4] = scales.to(device)
    got = ep.experts_linear(ep.Fp8Rows(wide[:, :256].view(torch.float8_e4m3fn), wide_scales[:, 2:4]), on(device, weight),
                            offsets.to(device), counts.to(device))
    close(got, z, slack)


@pytest.mark.parametrize("kernel", KERNELS)
def test_products_keep_a_nan_to_its_row_and_its_expert(device, tuning, kernel):
    tuning("EXPERTS_TILE", kernel)
    values, scales, weight, offsets, counts = make_product("uneven", 256, 256, 4)
    values.view(torch.uint8)[10, 77] = NAN_BYTE
    weight.values.view(torch.uint8)[3, 20, 100] = NAN_BYTE
    rows, weight = ep.Fp8Rows(values.to(device), scales.to(device)), on(device, weight)
    bad = torch.zeros(values.shape[0], 256, dtype=torch.bool)
    bad[10] = True
    bad[offsets[3] : offsets[3] + counts[3], 20] = True
    assert torch.equal(ep.experts_linear(rows, weight, offsets.to(device), counts.to(device)).cpu().isnan(), bad)
    got = ep.experts_gated(rows, weight, offsets.to(device), counts.to(device))
    reached = bad[:, :128] | bad[:, 128:]
    assert torch.equal(got.scales.cpu()[:, 0].isnan(), reached.any(1))


@pytest.mark.parametrize("kernel", KERNELS)
def test_products_stay_within_the_rows_whatever_the_layout_says(device, tuning, kernel):
    tuning("EXPERTS_TILE", kernel)
    values, scales = oracle.quantize_rows(randn(3, 64, 128))
    weight = ep.quantize_weight(randn(4, 3, 64, 128))
    rows = ep.Fp8Rows(values.to(device), scales.to(device))
    # an expert's count reaches past its segment, the last segment past the rows
    offsets, counts = torch.tensor([0, 20, 40, 90], device=device), torch.tensor([25, 20, 1 << 40], device=device)
    z, slack = oracle.experts(values, scales, weight.values, weight.scales, torch.tensor([0, 20, 40]), torch.tensor([20, 20, 24]))
    close(ep.experts_linear(rows, on(device, weight), offsets, counts), z, slack)


def test_products_of_no_rows(device):
    weight = on(device, ep.quantize_weight(randn(4, 3, 64, 128)))
    rows = ep.Fp8Rows(torch.empty(0, 128, dtype=torch.float8_e4m3fn, device=device), torch.empty(0, 1, device=device))
    offsets, counts = torch.zeros(4, dtype=torch.int64, device=device), torch.zeros(3, dtype=torch.int64, device=device)
    assert ep.experts_linear(rows, weight, offsets, counts).shape == (0, 64)
    assert ep.experts_gated(rows, weight, offsets, counts).values.shape == (0, 32)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12])
def test_products_of_small_and_large_scales(device, scale):
    values, scales, weight, offsets, counts = make_product("small", 256, 64, 5)
    scales = scales * scale
    z, slack = oracle.experts(values, scales, weight.values, weight.scales, offsets, counts)
    got = ep.experts_linear(ep.Fp8Rows(values.to(device), scales.to(device)), on(device, weight), offsets.to(device), counts.to(device))
    close(got, z, slack)


def test_products_of_rows_beyond_32_bit_offsets(device):
    # 2.4 GB of values: the last rows' offsets exceed 2^31 bytes, those of the output as well
    rows, inner, columns = 600_000, 4096, 2048
    values = torch.randint(0, 0x70, (rows, inner), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    scales = torch.rand(rows, inner // 128, device=device)
    weight = ep.quantize_weight(randn(6, 2, columns, inner))
    offsets = torch.tensor([0, rows - 100, rows], device=device)
    counts = torch.tensor([rows - 100, 100], device=device)
    got = ep.experts_linear(ep.Fp8Rows(values, scales), on(device, weight), offsets, counts)
    for e, part in ((0, slice(0, 40)), (0, slice(rows - 140, rows - 100)), (1, slice(rows - 100, rows))):
        z, slack = oracle.experts(values[part].cpu(), scales[part].cpu(), weight.values[e : e + 1], weight.scales[e : e + 1], None, None)
        close(got[part], z, slack)


def test_products_of_more_tiles_than_a_workgroup_lists(device):
    # 66000 tiles of 256 rows; whole numbers, whose products and sums are exact whatever adds them
    rows, inner, columns = 66_000 * 256 + 17, 128, 8
    whole = torch.randint(-4, 5, (rows, inner), dtype=torch.int8, device=device)
    values = torch.empty(rows, inner, dtype=torch.float8_e4m3fn, device=device)
    for part in range(0, rows, 1 << 20):
        values[part : part + (1 << 20)] = whole[part : part + (1 << 20)].to(torch.float8_e4m3fn)
    scales = 2.0 ** torch.randint(-3, 4, (rows, 1), device=device)
    weight = torch.randint(-4, 5, (1, columns, inner), generator=torch.Generator().manual_seed(6)).float()
    got = ep.experts_linear(ep.Fp8Rows(values, scales), ep.Fp8Weight(weight.to(torch.float8_e4m3fn).to(device), torch.ones(1, 1, 1, device=device)))
    for part in range(0, rows, 1 << 20):
        z = (whole[part : part + (1 << 20)].float() @ weight[0].T.to(device)) * scales[part : part + (1 << 20)]
        assert torch.equal(got[part : part + (1 << 20)], z.to(torch.bfloat16))


# ------------------------------------------------------------------ weighted combine


def make_weighted(tokens, topk, hidden, seed, spare=5):
    """Slots in no order, a fifth of the choices masked, one token without any; rows nobody names hold NaN."""
    generator = torch.Generator().manual_seed(seed)
    masked = torch.rand(tokens, topk, generator=generator) < 0.2
    if tokens > 1:
        masked[tokens // 2] = True
    rows = tokens * topk + spare
    slots = torch.randperm(rows, generator=generator)[: tokens * topk].reshape(tokens, topk).to(torch.int32)
    # both ways of naming no row
    slots[masked] = torch.where(torch.rand(int(masked.sum()), generator=generator) < 0.5, -1, rows + 3).to(torch.int32)
    y = randn(seed + 1, rows, hidden).to(torch.bfloat16)
    named = torch.zeros(rows, dtype=torch.bool)
    named[slots[~masked].long()] = True
    y[~named] = float("nan")
    weights = randn(seed + 2, tokens, topk)
    weights[masked] = float("nan")
    return y, slots, weights, named


WEIGHTED = [(1, 1, 8), (1, 8, 7168), (3, 2, 72), (129, 3, 1024), (40, 9, 520), (20, 32, 512), (257, 6, 2816), (300, 8, 1032)]


@pytest.mark.parametrize("tokens,topk,hidden", WEIGHTED)
@pytest.mark.parametrize("with_bias", [False, True])
def test_combine_weighted(device, tokens, topk, hidden, with_bias):
    y, slots, weights, _ = make_weighted(tokens, topk, hidden, tokens + hidden)
    bias = randn(8, tokens, hidden).to(torch.bfloat16) if with_bias else None
    out, slack = oracle.combine(y, slots, weights, bias)
    print("combine_weighted", tokens, topk, hidden, with_bias, flush=True)
    got = ep.combine_weighted(y.to(device), slots.to(device), weights.to(device), bias=None if bias is None else bias.to(device))
    close(got, out, slack)


@pytest.mark.parametrize("tokens,topk,hidden", WEIGHTED)
def test_combine_weighted_backward(device, tokens, topk, hidden):
    y, slots, weights, named = make_weighted(tokens, topk, hidden, tokens + hidden)
    grad = randn(9, tokens, hidden).to(torch.bfloat16)
    want_y, want_weights, slack = oracle.combine_backward(grad, y, slots, weights)
    print("combine_weighted_backward", tokens, topk, hidden, flush=True)
    grad_y, grad_weights = ep.combine_weighted_backward(grad.to(device), y.to(device), slots.to(device), weights.to(device))
    close(grad_y, want_y, want_y.abs() * oracle.FP32)
    assert not grad_y.cpu()[~named].any()
    assert ((grad_weights.cpu().double() - want_weights).abs() <= slack).all()


@pytest.mark.parametrize("alignment", [1, 16, 128])
def test_combine_weighted_backward_clears_the_rows_of_no_expert(device, alignment):
    tokens, topk, hidden, experts = 200, 4, 264, 12
    idx = torch.rand(tokens, experts, generator=torch.Generator().manual_seed(1)).topk(topk, dim=1).indices
    idx[idx == 5] = -1
    config = ep.EPConfig(experts, topk, 256, tokens)
    with ep.Buffer(None, config) as buffer:
        received = buffer.dispatch(torch.zeros(tokens, 256, dtype=torch.bfloat16, device=device), topk_idx=idx.to(device), do_expand=True,
                                   alignment=alignment)
    handle = received.handle
    rows = handle.layout.expanded_capacity + 9
    y, grad = randn(2, rows, hidden).to(torch.bfloat16), randn(3, tokens, hidden).to(torch.bfloat16)
    weights = torch.rand(tokens, topk)
    want_y, want_weights, slack = oracle.combine_backward(grad, y, handle.token_slots.cpu(), weights)
    torch.full((rows, hidden), float("nan"), dtype=torch.bfloat16, device=device)  # what a new tensor's memory may hold
    got = ep.combine_weighted_backward(grad.to(device), y.to(device), handle.token_slots, weights.to(device), handle.layout.expert_offsets,
                                       handle.layout.expert_counts)
    close(got[0], want_y, want_y.abs() * oracle.FP32)
    assert ((got[1].cpu().double() - want_weights).abs() <= slack).all()
    # the same without the layout, bit for bit
    again = ep.combine_weighted_backward(grad.to(device), y.to(device), handle.token_slots, weights.to(device))
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_the_gradient_is_the_difference(device):
    """The combine is linear in y and in the weights: with small whole numbers every difference is exact in bf16."""
    generator = torch.Generator().manual_seed(11)
    tokens, topk, hidden = 50, 3, 40

    def whole(*shape):
        return torch.randint(-3, 4, shape, generator=generator)

    slots = torch.randperm(tokens * topk, generator=generator).reshape(tokens, topk).to(torch.int32)
    slots[whole(tokens, topk) == 3] = -1
    y, dy = whole(tokens * topk, hidden).to(torch.bfloat16), whole(tokens * topk, hidden).to(torch.bfloat16)
    weights, dw, grad = whole(tokens, topk).float(), whole(tokens, topk).float(), whole(tokens, hidden).to(torch.bfloat16)
    at = [t.to(device) for t in (y, slots, weights, grad)]
    base = ep.combine_weighted(at[0], at[1], at[2]).double()
    along_y = (ep.combine_weighted(at[0] + dy.to(device), at[1], at[2]).double() - base) * at[3].double()
    along_weights = (ep.combine_weighted(at[0], at[1], at[2] + dw.to(device)).double() - base) * at[3].double()
    grad_y, grad_weights = ep.combine_weighted_backward(at[3], at[0], at[1], at[2])
    assert along_y.sum() == (grad_y.double() * dy.to(device).double()).sum()
    assert along_weights.sum() == (grad_weights.double() * dw.to(device).double()).sum()


def test_autograd_from_the_source_rows_to_the_output(device):
    """dispatch_rows -> experts in torch -> combine_weighted, against the dense layer in 64 bits."""
    tokens, topk, hidden, experts = 60, 3, 256, 5
    idx = torch.rand(tokens, experts, generator=torch.Generator().manual_seed(2)).topk(topk, dim=1).indices
    idx[7] = -1
    x, gain = randn(1, tokens, hidden).to(torch.bfloat16), (1 + 0.2 * randn(2, experts, hidden)).to(torch.bfloat16)
    weights, bias = torch.rand(tokens, topk), randn(4, tokens, hidden).to(torch.bfloat16)
    grad = randn(5, tokens, hidden).to(torch.bfloat16)
    with ep.Buffer(None, ep.EPConfig(experts, topk, hidden, tokens)) as buffer:
        handle = buffer.dispatch(x.to(device), topk_idx=idx.to(device), do_expand=True, alignment=8).handle
        layout = handle.layout
        xs, ws, bs, gains = (t.to(device).requires_grad_() for t in (x, weights, bias, gain))
        rows = ep.dispatch_rows(buffer, xs, handle)
        expert = torch.searchsorted(layout.expert_offsets[1:].contiguous(), torch.arange(rows.shape[0], device=device), right=True)
        out = ep.combine_weighted(rows * gains[expert], handle.token_slots, ws, bias=bs, expert_offsets=layout.expert_offsets,
                                  expert_counts=layout.expert_counts)
        out.backward(grad.to(device))
    dense = [t.double().requires_grad_() for t in (x, weights, bias, gain)]
    chosen = (idx >= 0)[:, :, None]
    want = dense[2] + (dense[0][:, None] * dense[3][idx.clamp(min=0)] * dense[1][:, :, None] * chosen).sum(1)
    want.backward(grad.double())
    # every step rounds to bf16 once, and a source row's gradient adds three such rows; whole-tensor norms
    for got, exact in zip((out, xs.grad, ws.grad, bs.grad, gains.grad), (want, *(t.grad for t in dense))):
        assert (got.detach().cpu().double() - exact).norm() <= 4 * oracle.BF16 * exact.norm()


def test_autograd_gives_only_the_gradients_that_are_asked_for(device):
    y, slots, weights, _ = make_weighted(10, 2, 64, 3)
    y = torch.nan_to_num(y)
    at = [t.to(device) for t in (y, slots, torch.nan_to_num(weights))]
    bias = torch.zeros(10, 64, dtype=torch.bfloat16, device=device, requires_grad=True)
    ep.combine_weighted(*at, bias=bias).sum().backward()
    assert (bias.grad == 1).all()
    ws = at[2].clone().requires_grad_()
    ep.combine_weighted(at[0], at[1], ws).sum().backward()
    assert ws.grad.shape == ws.shape
    with torch.no_grad():
        assert not ep.combine_weighted(at[0], at[1], ws).requires_grad


def test_weighted_rows_beyond_32_bit_offsets(device):
    rows, hidden, tokens = 300_000, 7168, 64
    y = torch.zeros(rows, hidden, dtype=torch.bfloat16, device=device)
    slots = torch.randperm(rows, generator=torch.Generator().manual_seed(3))[: tokens * 2].reshape(tokens, 2).to(torch.int32)
    slots[0, 0], slots[1, 1] = rows - 1, rows - 2
    named = slots.flatten().long()
    y[named.to(device)] = randn(1, tokens * 2, hidden).to(torch.bfloat16).to(device)
    few, dense_slots = y[named.to(device)].cpu(), torch.arange(tokens * 2, dtype=torch.int32).reshape(tokens, 2)
    weights, grad = torch.rand(tokens, 2), randn(4, tokens, hidden).to(torch.bfloat16)
    close(ep.combine_weighted(y, slots.to(device), weights.to(device)), *oracle.combine(few, dense_slots, weights, None))
    grad_y, grad_weights = ep.combine_weighted_backward(grad.to(device), y, slots.to(device), weights.to(device))
    want_y, want_weights, slack = oracle.combine_backward(grad, few, dense_slots, weights)
    close(grad_y[named.to(device)], want_y, want_y.abs() * oracle.FP32)
    assert ((grad_weights.cpu().double() - want_weights).abs() <= slack).all()


# ------------------------------------------------------------------ streams, graphs, refusals


def test_operators_run_on_the_current_stream(device):
    """Behind work of the same stream, while the default stream has nothing of it."""
    side = torch.cuda.Stream()
    values, scales, weight, offsets, counts = make_product("uneven", 256, 256, 4)
    want = ep.experts_linear(ep.Fp8Rows(values.to(device), scales.to(device)), on(device, weight), offsets.to(device), counts.to(device))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        busy = torch.zeros(1 << 26, device=device)
        for _ in range(20):
            busy += 1
        rows = ep.Fp8Rows(values.to(device), scales.to(device))
        got = ep.experts_linear(rows, on(device, weight), offsets.to(device), counts.to(device))
    side.synchronize()
    assert torch.equal(got, want)


def test_a_captured_layer_replays(device):
    tokens, topk, hidden, experts = 24, 2, 256, 4
    gamma = torch.ones(hidden, dtype=torch.bfloat16, device=device)
    idx = torch.rand(tokens, experts, generator=torch.Generator().manual_seed(4)).topk(topk, dim=1).indices.to(device)
    weights = torch.rand(tokens, topk, device=device)
    gate_up, down = (on(device, ep.quantize_weight(randn(s, experts, c, hidden) / 16)) for s, c in ((1, 512), (2, 256)))
    x = torch.zeros(tokens, hidden, dtype=torch.bfloat16, device=device)
    with ep.Buffer(None, ep.EPConfig(experts, topk, ep.fp8_payload_width(hidden), tokens)) as buffer:
        payload = ep.rms_norm_fp8(x, gamma).rows.payload
        handle = buffer.dispatch(payload, topk_idx=idx, do_expand=True, alignment=4).handle
        segments = (handle.layout.expert_offsets, handle.layout.expert_counts)

        def layer():
            received = buffer.dispatch(ep.rms_norm_fp8(x, gamma).rows.payload, handle=handle, zero_padding=True)
            act = ep.experts_gated(ep.Fp8Rows.of_payload(received.x, hidden), gate_up, *segments)
            y = ep.experts_linear(act, down, *segments)
            out = ep.combine_weighted(y, handle.token_slots, weights, bias=x)
            return out, *ep.combine_weighted_backward(out, y, handle.token_slots, weights, *segments)

        layer()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = layer()
        for step in range(4):
            x.copy_(randn(step, tokens, hidden))
            graph.replay()
            replayed = [t.clone() for t in captured]
            for got, want in zip(replayed, layer()):
                assert torch.equal(got, want)
            torch.cuda.synchronize()


def test_refusals(device):
    bf16 = dict(dtype=torch.bfloat16, device=device)
    x, gamma = torch.zeros(4, 256, **bf16), torch.ones(256, **bf16)
    rows, weight = ep.rms_norm_fp8(x, gamma).rows, on(device, ep.quantize_weight(randn(1, 2, 64, 256)))
    offsets, counts = torch.tensor([0, 2, 4], device=device), torch.tensor([2, 2], device=device)
    slots, weights = torch.zeros(4, 1, dtype=torch.int32, device=device), torch.ones(4, 1, device=device)
    shifted = torch.zeros(4 * 256 + 4, **bf16)[4:].view(4, 256)
    refused = [
        lambda: ep.rms_norm_fp8(x.cpu(), gamma),
        lambda: ep.rms_norm_fp8(x.float(), gamma),
        lambda: ep.rms_norm_fp8(x[0], gamma),
        lambda: ep.rms_norm_fp8(x[:, ::2], gamma[:128]),
        lambda: ep.rms_norm_fp8(x[:, :250].contiguous(), gamma[:250]),
        lambda: ep.rms_norm_fp8(x, gamma.float()),
        lambda: ep.rms_norm_fp8(x, gamma, residual=x[:3]),
        lambda: ep.rms_norm_fp8(x, gamma, eps=-1.0),
        lambda: ep.rms_norm_fp8(x, gamma, eps=float("nan")),
        lambda: ep.rms_norm_fp8(shifted, gamma),
        lambda: ep.experts_linear(rows, weight),
        lambda: ep.experts_linear(rows, weight, offsets),
        lambda: ep.experts_linear(rows, weight, offsets[:2], counts),
        lambda: ep.experts_linear(rows, weight, offsets.int(), counts),
        lambda: ep.experts_linear(rows, weight, offsets.cpu(), counts),
        lambda: ep.experts_linear(ep.Fp8Rows(x, rows.scales), weight, offsets, counts),
        lambda: ep.experts_linear(ep.Fp8Rows(rows.values, rows.scales[:, :1]), weight, offsets, counts),
        lambda: ep.experts_linear(ep.Fp8Rows(rows.values, rows.scales.double()), weight, offsets, counts),
        lambda: ep.experts_linear(ep.Fp8Rows(rows.values[:, :248], rows.scales), weight, offsets, counts),
        lambda: ep.experts_linear(rows, ep.Fp8Weight(weight.values[:, :60], weight.scales), offsets, counts),
        lambda: ep.experts_linear(rows, ep.Fp8Weight(weight.values.transpose(1, 2), weight.scales), offsets, counts),
        lambda: ep.experts_linear(rows, ep.Fp8Weight(weight.values, weight.scales[:1]), offsets, counts),
        lambda: ep.experts_gated(rows, ep.Fp8Weight(weight.values[:, :48].contiguous(), weight.scales), offsets, counts),
        lambda: ep.combine_weighted(x.float(), slots, weights),
        lambda: ep.combine_weighted(x, slots.long(), weights),
        lambda: ep.combine_weighted(x, slots, weights.double()),
        lambda: ep.combine_weighted(x, slots, weights[:3]),
        lambda: ep.combine_weighted(x, slots, weights, bias=x[:3]),
        lambda: ep.combine_weighted(x[:, :252].contiguous(), slots, weights),
        lambda: ep.combine_weighted(shifted, slots, weights),
        lambda: ep.combine_weighted(x, slots.expand(4, 33).contiguous(), weights.expand(4, 33).contiguous()),
        lambda: ep.combine_weighted_backward(x[:3], x, slots, weights),
        lambda: ep.combine_weighted_backward(x, x, slots, weights, offsets),
        lambda: ep.combine_weighted_backward(x, x, slots, weights, offsets, counts[:1]),
        lambda: ep.Fp8Rows.of_payload(x, 1024),
        lambda: ep.fp8_payload_width(250),
        lambda: ep.quantize_weight(x),
    ]
    for n, call in enumerate(refused):
        print("refusal", n, flush=True)
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="has no gradient"):
        ep.rms_norm_fp8(x.clone().requires_grad_(), gamma)
    with torch.no_grad():
        ep.rms_norm_fp8(x.clone().requires_grad_(), gamma)
