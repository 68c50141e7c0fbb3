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
