"""What of the operators' edges needs no GPU."""

import inspect
import re

import pytest
import torch

import nanoep_amd as ep
from nanoep_amd import operators
from nanoep_amd.build import CSRC
from test_operators_host import library


@pytest.mark.parametrize("columns", [(1 << 24) + 32, 1 << 30])
def test_more_columns_than_the_products_take_are_refused(columns):
    lib, null = library(), None
    assert lib.nanoep_experts_linear(64, 128, 64, 1, 64, 64, null, null, 1, 1, 128, columns, 64, null) == 1
    assert lib.nanoep_experts_gated(64, 128, 64, 1, 64, 64, null, null, 1, 1, 128, columns, 64, 64, 1 << 40, null) == 1


def test_statements_that_write_m0_say_so():
    """An assembly statement whose clobbers leave out a register that it writes is right only while nobody else uses it."""
    found = 0
    for source in sorted(CSRC.glob("*")):
        for statement in re.findall(r"\basm\b[^;]*?;", re.sub(r"//[^\n]*", "", source.read_text()), re.S):
            if re.search(r"\bm0\s*,", statement.split(":")[0]):
                found += 1
                assert '"m0"' in statement.split(":")[-1], f"{source.name}: {statement}"
    assert found == 4


def test_every_function_that_the_operators_bind_is_called():
    bound = set(re.findall(r'module\.def\("(\w+)"', (CSRC / "nanoep_operators.cpp").read_text()))
    called = set(re.findall(r"load_extension\(\)\.(\w+)\(", inspect.getsource(operators)))
    assert bound == called


def test_records_that_start_between_two_scales_are_refused():
    width = ep.fp8_payload_width(256)
    storage = torch.zeros(3 * width + 2, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ep.Fp8Rows.of_payload(storage[1 : 1 + 3 * width].view(3, width), 256)
    assert ep.Fp8Rows.of_payload(storage[2:].view(3, width), 256).scales.shape == (3, 2)
