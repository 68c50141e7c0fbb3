"""The expert layer's operators where ordinary inputs do not lead: products that cancel, sizes at the ends of what is taken,
gradients that arrive in unusual tensors, derivatives that do not exist."""

import pytest
import torch

import nanoep_amd as ep
import operator_oracle as oracle
from test_gpu_operators import KERNELS, close, on

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
