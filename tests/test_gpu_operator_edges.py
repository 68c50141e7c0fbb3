"""The expert layer's operators where ordinary inputs do not lead: products that cancel, sizes at the ends of what is taken,
gradients that arrive in unusual tensors, derivatives that do not exist."""

import pytest
import torch
from torch.autograd import forward_ad

import nanoep_amd as ep
import operator_oracle as oracle
from test_gpu_operators import KERNELS, NAN_BYTE, close, make_product, on, randn

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ products


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("inner", [16, 128, 272, 640])
def test_products_of_terms_that_cancel(device, tuning, inner, kernel):
    """Two products of a block are 448 * 448 and its negative, the others 1 to 3: sums of whole numbers below 2^24, each of them exact
    in fp32."""
    tuning("EXPERTS_TILE", kernel)
    counts, columns = torch.tensor([3, 0, 70, 130]), 96
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    rows = int(offsets[-1])
    values = torch.randint(1, 4, (rows, inner), generator=torch.Generator().manual_seed(inner)).float()
    first, second = inner - 13, inner - 4  # both in the last block
    values[:, first], values[:, second] = 448.0, -448.0
    values[1::2, [first, second]] *= -1.0
    weight = torch.ones(len(counts), columns, inner)
    weight[:, :, [first, second]] = 448.0
    values, weight = values.to(torch.float8_e4m3fn), weight.to(torch.float8_e4m3fn)
    scales = torch.full((rows, oracle.groups(inner)), 2.0**-8)
    weight = ep.Fp8Weight(weight, torch.ones(len(counts), 1, oracle.groups(inner)))
    z, slack = oracle.experts(values, scales, weight.values, weight.scales, offsets, counts)
    assert slack.max() < z.min() / 4  # a sum that loses the small products is out of it
    layout = (offsets.to(device), counts.to(device))
    on_device = ep.Fp8Rows(values.to(device), scales.to(device))
    print("products that cancel", inner, kernel, flush=True)
    close(ep.experts_linear(on_device, on(device, weight), *layout), z, slack)
    got = ep.experts_gated(on_device, on(device, weight), *layout)
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), *oracle.gated(z, slack))


@pytest.mark.parametrize("columns", [(1 << 21) + 32, 1 << 24])
def test_products_of_more_columns_than_a_grid_axis_has_steps(device, columns):
    """Whole numbers: every product and sum is exact.  A row behind the expert's, and one behind the last segment."""
    generator = torch.Generator().manual_seed(columns)
    inner, rows = 16, 5
    layout = torch.tensor([0, 4], device=device), torch.tensor([3], device=device)
    values = torch.randint(-4, 5, (rows, inner), generator=generator).float()
    weight = torch.randint(-4, 5, (1, columns, inner), generator=generator, dtype=torch.int8).float()
    rows_on = ep.Fp8Rows(values.to(torch.float8_e4m3fn).to(device), torch.ones(rows, 1, device=device))
    weight_on = ep.Fp8Weight(weight.to(torch.float8_e4m3fn).to(device), torch.ones(1, oracle.groups(columns), 1, device=device))
    z = values @ weight[0].T
    z[3:] = 0
    print("columns", columns, flush=True)
    assert torch.equal(ep.experts_linear(rows_on, weight_on, *layout).cpu(), z.to(torch.bfloat16))
    got = ep.experts_gated(rows_on, weight_on, *layout)
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), *oracle.gated(z.double(), torch.zeros_like(z).double()))


def test_products_of_more_row_tiles_than_a_grid_axis_has_threads_for(device, tuning):
    """2^24 tiles of 64 rows, of 256 threads each; the same whole numbers over and over, in a period that no grid has."""
    tuning("EXPERTS_TILE", 1)
    period, inner, columns = 4_000_037, 16, 8
    rows = (1 << 30) + 70
    whole = torch.randint(-4, 5, (period, inner), device=device).float()
    weight = torch.randint(-4, 5, (1, columns, inner), generator=torch.Generator().manual_seed(6)).float()
    values = torch.empty(rows, inner, dtype=torch.float8_e4m3fn, device=device)
    for part in range(0, rows, period):
        values[part : part + period] = whole[: rows - part].to(torch.float8_e4m3fn)
    scales = torch.ones(rows, 1, device=device)
    want = (whole @ weight[0].T.to(device)).to(torch.bfloat16)
    layout = torch.tensor([0, rows - 3], device=device), torch.tensor([rows - 5], device=device)
    print("row tiles", rows, flush=True)
    got = ep.experts_linear(ep.Fp8Rows(values, scales), ep.Fp8Weight(weight.to(torch.float8_e4m3fn).to(device), torch.ones(1, 1, 1, device=device)), *layout)
    assert not got[rows - 5 :].any()
    for part in range(0, rows - 5, period):
        assert torch.equal(got[part : min(part + period, rows - 5)], want[: rows - 5 - part])


@pytest.mark.parametrize("kernel", KERNELS)
def test_products_of_segments_that_lie_over_one_another(device, tuning, kernel):
    """Every other segment is all rows, which have tiles for two of them; the experts' weights are the same."""
    tuning("EXPERTS_TILE", kernel)
    experts, rows = 2000, 1000
    values, scales = oracle.quantize_rows(randn(3, rows, 128))
    weight = ep.quantize_weight(randn(4, 1, 64, 128))
    weight = ep.Fp8Weight(weight.values.expand(experts, -1, -1).contiguous(), weight.scales.expand(experts, -1, -1).contiguous())
    offsets = torch.tensor([0, rows] * (experts // 2) + [rows], device=device)
    counts = torch.full((experts,), rows, device=device)
    z, slack = oracle.experts(values, scales, weight.values[:1], weight.scales[:1], None, None)
    rows_on, weight = ep.Fp8Rows(values.to(device), scales.to(device)), on(device, weight)
    print("segments over one another", kernel, flush=True)
    close(ep.experts_linear(rows_on, weight, offsets, counts), z, slack)
    got = ep.experts_gated(rows_on, weight, offsets, counts)
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), *oracle.gated(z, slack))


@pytest.mark.parametrize("kernel", KERNELS)
def test_gated_products_follow_strides_of_their_own(device, tuning, kernel):
    tuning("EXPERTS_TILE", kernel)
    values, scales, weight, offsets, counts = make_product("uneven", 272, 160, 9)
    rows = values.shape[0]
    wide = torch.full((rows, 272 + 48), NAN_BYTE, dtype=torch.uint8, device=device)
    wide[:, 16:288] = values.view(torch.uint8).to(device)
    wide_scales = torch.full((rows, 7), float("nan"), device=device)
    wide_scales[:, 2:5] = scales.to(device)
    print("gated strides", kernel, flush=True)
    got = ep.experts_gated(ep.Fp8Rows(wide[:, 16:288].view(torch.float8_e4m3fn), wide_scales[:, 2:5]), on(device, weight), offsets.to(device),
                           counts.to(device))
    z = oracle.experts(values, scales, weight.values, weight.scales, offsets, counts)
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), *oracle.gated(*z))


@pytest.mark.parametrize("kernel", KERNELS)
def test_gated_products_stay_within_the_rows_whatever_the_layout_says(device, tuning, kernel):
    tuning("EXPERTS_TILE", kernel)
    values, scales = oracle.quantize_rows(randn(3, 64, 128))
    weight = ep.quantize_weight(randn(4, 3, 64, 128))
    # an expert's count reaches past its segment, the last segment past the rows
    offsets, counts = torch.tensor([0, 20, 40, 90], device=device), torch.tensor([25, 20, 1 << 40], device=device)
    z = oracle.experts(values, scales, weight.values, weight.scales, torch.tensor([0, 20, 40]), torch.tensor([20, 20, 24]))
    print("gated layout", kernel, flush=True)
    got = ep.experts_gated(ep.Fp8Rows(values.to(device), scales.to(device)), on(device, weight), offsets, counts)
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), *oracle.gated(*z))


def test_gated_products_of_rows_beyond_32_bit_offsets(device):
    rows, inner, columns = 600_000, 4096, 64
    values = torch.randint(0, 0x70, (rows, inner), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    scales = torch.rand(rows, inner // 128, device=device) * 1e-3
    weight = ep.quantize_weight(randn(6, 2, columns, inner))
    layout = torch.tensor([0, rows - 100, rows], device=device), torch.tensor([rows - 100, 100], device=device)
    got = ep.experts_gated(ep.Fp8Rows(values, scales), on(device, weight), *layout)
    for e, part in ((0, slice(0, 40)), (0, slice(rows - 140, rows - 100)), (1, slice(rows - 100, rows))):
        z = oracle.experts(values[part].cpu(), scales[part].cpu(), weight.values[e : e + 1], weight.scales[e : e + 1], None, None)
        oracle.check_eight_bits(got.values[part].cpu(), got.scales[part].cpu(), *oracle.gated(*z))


def test_gated_products_of_more_tiles_than_a_workgroup_lists(device, tuning):
    """66000 tiles of 256 rows; whole numbers, whose sums are exact."""
    tuning("EXPERTS_TILE", 256)
    rows, inner, columns = 66_000 * 256 + 17, 16, 32
    whole = torch.randint(-4, 5, (rows, inner), dtype=torch.int8, device=device)
    scales = 2.0 ** torch.randint(-3, 4, (rows, 1), device=device)
    weight = torch.randint(-4, 5, (1, columns, inner), generator=torch.Generator().manual_seed(6)).float()
    weight_on = ep.Fp8Weight(weight.to(torch.float8_e4m3fn).to(device), torch.ones(1, 1, 1, device=device))
    print("gated tiles", rows, flush=True)
    got = ep.experts_gated(ep.Fp8Rows(whole.to(torch.float8_e4m3fn), scales), weight_on)
    for part in range(0, rows, 1 << 20):
        at = slice(part, part + (1 << 20))
        z = ((whole[at].float() @ weight[0].T.to(device)) * scales[at]).double()
        oracle.check_eight_bits(got.values[at], got.scales[at], *oracle.gated(z, torch.zeros_like(z)))


def test_products_with_an_experts_weight_beyond_32_bit_offsets(device):
    inner, columns, rows = 4112, (1 << 20) + 256, 3
    assert inner * columns > 1 << 32
    values, scales = oracle.quantize_rows(randn(1, rows, inner))
    weight = torch.randint(0, 0x70, (1, columns, inner), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    weight_scales = torch.rand(1, oracle.groups(columns), oracle.groups(inner), device=device) * 1e-3
    rows_on, weight_on = ep.Fp8Rows(values.to(device), scales.to(device)), ep.Fp8Weight(weight, weight_scales)
    print("weight beyond 32 bits", flush=True)
    linear, gated = ep.experts_linear(rows_on, weight_on), ep.experts_gated(rows_on, weight_on)

    def z_of(part):
        blocks = slice(part.start // 128, part.stop // 128)
        return oracle.experts(values, scales, weight[:, part].cpu(), weight_scales[:, blocks].cpu(), None, None)

    half = columns // 2
    for begin in (0, half - 128 * 5, half - 128):
        part, above = slice(begin, begin + 128), slice(half + begin, half + begin + 128)
        (gate, gate_slack), (up, up_slack) = z_of(part), z_of(above)
        close(linear[:, part], gate, gate_slack)
        close(linear[:, above], up, up_slack)
        act = oracle.gated(torch.cat([gate, up], 1), torch.cat([gate_slack, up_slack], 1))
        oracle.check_eight_bits(gated.values[:, part].cpu(), gated.scales[:, begin // 128 : begin // 128 + 1].cpu(), *act)


def test_products_of_more_experts_than_a_tile_list_takes(device):
    experts, inner, columns = (1 << 14) + 3, 32, 64
    counts = torch.randint(0, 3, (experts,), generator=torch.Generator().manual_seed(2))
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), ((counts + 3) // 4 * 4).cumsum(0)])
    rows = int(offsets[-1]) + 2
    values, scales = oracle.quantize_rows(randn(3, rows, inner))
    weight = randn(4, experts, columns, inner).clamp(-4, 4).mul(100).to(torch.float8_e4m3fn)
    weight_scales = torch.rand(experts, 1, 1) * 1e-2
    z = oracle.experts(values, scales, weight, weight_scales, offsets, counts)
    rows_on, weight_on = ep.Fp8Rows(values.to(device), scales.to(device)), on(device, ep.Fp8Weight(weight, weight_scales))
    print("experts", experts, flush=True)
    close(ep.experts_linear(rows_on, weight_on, offsets.to(device), counts.to(device)), *z)
    got = ep.experts_gated(rows_on, weight_on, offsets.to(device), counts.to(device))
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), *oracle.gated(*z))


@pytest.mark.parametrize("value_stride,scale_stride", [((1 << 24) + 16, 3), (272, (1 << 22) + 1)])
def test_products_of_rows_far_apart(device, value_stride, scale_stride):
    rows, inner, columns = 70, 272, 96
    values, scales = oracle.quantize_rows(randn(5, rows, inner))
    weight = ep.quantize_weight(randn(6, 1, columns, inner))
    far = torch.full((rows * value_stride,), NAN_BYTE, dtype=torch.uint8, device=device).view(rows, value_stride)[:, :inner].view(torch.float8_e4m3fn)
    far.view(torch.uint8).copy_(values.view(torch.uint8))
    far_scales = torch.full((rows * scale_stride,), float("nan"), device=device).view(rows, scale_stride)[:, :3]
    far_scales.copy_(scales)
    z = oracle.experts(values, scales, weight.values, weight.scales, None, None)
    print("rows apart", value_stride, scale_stride, flush=True)
    close(ep.experts_linear(ep.Fp8Rows(far, far_scales), on(device, weight)), *z)
    got = ep.experts_gated(ep.Fp8Rows(far, far_scales), on(device, weight))
    oracle.check_eight_bits(got.values.cpu(), got.scales.cpu(), *oracle.gated(*z))


# ------------------------------------------------------------------ norm and combine


def test_rms_norm_of_more_rows_than_a_grid_axis_has_threads_for(device):
    """2^26 rows, of 64 threads each."""
    period, tokens = 4_000_037, (1 << 26) + 5
    few = torch.randn(period, 16, device=device).to(torch.bfloat16)
    x = torch.empty(tokens, 16, dtype=torch.bfloat16, device=device)
    for part in range(0, tokens, period):
        x[part : part + period] = few[: tokens - part]
    gamma = torch.ones(16, dtype=torch.bfloat16, device=device)
    print("rms_norm_fp8", tokens, flush=True)
    got, want = ep.rms_norm_fp8(x, gamma).rows.payload.view(torch.int32), ep.rms_norm_fp8(few, gamma).rows.payload.view(torch.int32)
    for part in range(0, tokens, period):
        assert torch.equal(got[part : part + period], want[: tokens - part])


def test_combines_of_more_rows_than_a_grid_axis_has_threads_for(device):
    """2^24 workgroups of 256 threads: four tokens each, four choices each of the gradient."""
    generator = torch.Generator(device=device).manual_seed(7)
    tokens = (1 << 26) - 1
    y = torch.randn(1000, 8, device=device, generator=generator).to(torch.bfloat16)
    slots = torch.randint(-1, 1000, (tokens, 1), dtype=torch.int32, device=device, generator=generator)
    weights = torch.rand(tokens, 1, device=device, generator=generator)
    print("combine_weighted", tokens, flush=True)
    got = ep.combine_weighted(y, slots, weights)
    for part in range(0, tokens, 1 << 22):
        at = slice(part, part + (1 << 22))
        want = torch.where(slots[at] >= 0, y[slots[at, 0].clamp(min=0).long()].float() * weights[at], 0.0)
        assert torch.equal(got[at], want.to(torch.bfloat16))

    tokens, topk = (1 << 23) + 1, 8
    rows = tokens * topk
    y = torch.randn(rows, 8, device=device, generator=generator).to(torch.bfloat16)
    slots = torch.randperm(rows, device=device, generator=generator).to(torch.int32).reshape(tokens, topk)
    weights = torch.rand(tokens, topk, device=device, generator=generator)
    grad = torch.randn(tokens, 8, device=device, generator=generator).to(torch.bfloat16)
    print("combine_weighted_backward", tokens, flush=True)
    grad_y, grad_weights = ep.combine_weighted_backward(grad, y, slots, weights)
    for part in range(0, tokens, 1 << 20):
        at = slice(part, part + (1 << 20))
        g = grad[at, None].float()
        assert torch.equal(grad_y[slots[at].long()], (weights[at, :, None] * g).to(torch.bfloat16))
        terms = y[slots[at].long()].double() * g
        assert ((grad_weights[at].double() - terms.sum(2)).abs() <= terms.abs().sum(2) * oracle.FP32 * 8).all()


# ------------------------------------------------------------------ gradients


def test_gradients_that_arrive_off_their_alignment(device):
    """The gradient of a part of a concatenation is a contiguous view that starts anywhere."""
    tokens, topk, hidden, experts = 33, 2, 256, 4
    idx = torch.rand(tokens, experts, generator=torch.Generator().manual_seed(3)).topk(topk, dim=1).indices.to(device)
    x, weights = randn(1, tokens, hidden).to(torch.bfloat16).to(device), torch.rand(tokens, topk, device=device)
    bias = randn(2, tokens, hidden).to(torch.bfloat16).to(device)
    few = torch.zeros(3, dtype=torch.bfloat16, device=device)
    with ep.Buffer(None, ep.EPConfig(experts, topk, hidden, tokens)) as buffer:
        handle = buffer.dispatch(x, topk_idx=idx, do_expand=True, alignment=8).handle
        rows = ep.dispatch_rows(buffer, x, handle)
        grad = randn(4, 3 + tokens * hidden).to(torch.bfloat16).to(device)
        aligned = grad[3:].clone().view(tokens, hidden)

        leaves = [t.clone().requires_grad_() for t in (rows, weights, bias)]
        out = ep.combine_weighted(leaves[0], handle.token_slots, leaves[1], bias=leaves[2])
        torch.cat([few, out.flatten()]).backward(grad)
        want = ep.combine_weighted_backward(aligned, rows, handle.token_slots, weights)
        for leaf, gradient in zip(leaves, (*want, aligned)):
            assert torch.equal(leaf.grad, gradient)

        source = x.clone().requires_grad_()
        moved = ep.dispatch_rows(buffer, source, handle)
        grad = randn(5, 3 + moved.numel()).to(torch.bfloat16).to(device)
        torch.cat([few, moved.flatten()]).backward(grad)
        assert torch.equal(source.grad, buffer.combine(grad[3:].clone().view(moved.shape), handle).x)


def test_many_rows_of_no_expert_are_cleared_ahead_of_the_gradient(device):
    """More than 32 MiB of them have a launch of their own."""
    tokens, topk, hidden, experts = 50, 4, 2816, 128
    idx = torch.rand(tokens, experts, generator=torch.Generator().manual_seed(1)).topk(topk, dim=1).indices
    idx[idx % 7 == 0] = -1
    with ep.Buffer(None, ep.EPConfig(experts, topk, 256, tokens)) as buffer:
        handle = buffer.dispatch(torch.zeros(tokens, 256, dtype=torch.bfloat16, device=device), topk_idx=idx.to(device), do_expand=True,
                                 alignment=128).handle
    rows = handle.layout.expanded_capacity + 3
    assert (rows - tokens * topk) * hidden * 2 > 32 << 20
    y, grad = randn(2, rows, hidden).to(torch.bfloat16), randn(3, tokens, hidden).to(torch.bfloat16)
    weights = torch.rand(tokens, topk)
    want_y, want_weights, slack = oracle.combine_backward(grad, y, handle.token_slots.cpu(), weights)
    inputs = grad.to(device), y.to(device), handle.token_slots, weights.to(device)
    torch.full((rows, hidden), float("nan"), dtype=torch.bfloat16, device=device)  # what a new tensor's memory may hold
    got = ep.combine_weighted_backward(*inputs, handle.layout.expert_offsets, handle.layout.expert_counts)
    close(got[0], want_y, want_y.abs() * oracle.FP32)
    assert ((got[1].cpu().double() - want_weights).abs() <= slack).all()
    again = ep.combine_weighted_backward(*inputs)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_layouts_are_checked_ahead_of_the_combine(device):
    """Not in the backward pass, or never."""
    y, slots, weights = torch.zeros(4, 256, dtype=torch.bfloat16, device=device), torch.zeros(4, 1, dtype=torch.int32, device=device), torch.ones(4, 1, device=device)
    offsets, counts = torch.tensor([0, 2, 4], device=device), torch.tensor([2, 2], device=device)
    ep.combine_weighted(y, slots, weights, expert_offsets=offsets, expert_counts=counts)
    for layout in ((offsets, None), (None, counts), (offsets, counts[:1]), (offsets[:2], counts), (offsets.int(), counts), (offsets, counts.cpu()),
                   (offsets[:1], counts[:0])):
        for needed in (False, True):
            with pytest.raises(ValueError):
                ep.combine_weighted(y, slots, weights.clone().requires_grad_(needed), expert_offsets=layout[0], expert_counts=layout[1])


# ------------------------------------------------------------------ derivatives that the operators do not have


def calls_of_every_operator(device):
    """Name, call and its floating inputs."""
    y, slots, weights = torch.zeros(4, 256, dtype=torch.bfloat16, device=device), torch.arange(4, dtype=torch.int32, device=device)[:, None], torch.ones(4, 1, device=device)
    gamma = torch.ones(256, dtype=torch.bfloat16, device=device)
    rows, weight = ep.rms_norm_fp8(y, gamma).rows, on(device, ep.quantize_weight(randn(1, 1, 64, 256)))
    scales = rows.scales.contiguous()
    return [
        ("rms_norm_fp8", lambda x, g, r: ep.rms_norm_fp8(x, g, residual=r), (y, gamma, y.clone())),
        ("experts_linear", lambda s, w: ep.experts_linear(ep.Fp8Rows(rows.values, s), ep.Fp8Weight(weight.values, w)), (scales, weight.scales)),
        ("experts_gated", lambda s, w: ep.experts_gated(ep.Fp8Rows(rows.values, s), ep.Fp8Weight(weight.values, w)), (scales, weight.scales)),
        ("combine_weighted", lambda v, w, b: ep.combine_weighted(v, slots, w, bias=b), (y, weights, y.clone())),
        ("combine_weighted_backward", lambda g, v, w: ep.combine_weighted_backward(g, v, slots, w), (y, y.clone(), weights)),
    ]


def test_forward_mode_derivatives_are_refused(device):
    """A result without its tangent would pass for one that does not depend on the input."""
    for name, call, inputs in calls_of_every_operator(device):
        for which in range(len(inputs)):
            print("forward mode", name, which, flush=True)
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(inputs[which], torch.ones_like(inputs[which]))
                arguments = [*inputs[:which], dual, *inputs[which + 1 :]]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*arguments)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*arguments)
                call(*inputs)
    # beside an input that reverse mode follows, and through the functions that torch.autograd knows
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=device)
    idx = torch.arange(4, device=device)[:, None]
    with ep.Buffer(None, ep.EPConfig(4, 1, 256, 4)) as buffer, forward_ad.dual_level():
        handle = buffer.dispatch(x, topk_idx=idx, do_expand=True).handle
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError):
            ep.dispatch_rows(buffer, dual, handle)
        with pytest.raises(RuntimeError):
            ep.combine_weighted(dual, handle.token_slots, torch.ones(4, 1, device=device, requires_grad=True))


def test_the_gradients_own_gradient_is_refused(device):
    name, call, inputs = calls_of_every_operator(device)[-1]
    for which in range(len(inputs)):
        arguments = [*inputs[:which], inputs[which].clone().requires_grad_(), *inputs[which + 1 :]]
        with pytest.raises(RuntimeError, match="has no gradient"):
            call(*arguments)
        with torch.no_grad():
            call(*arguments)
