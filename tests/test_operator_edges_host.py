"""What of the operators' edges needs no GPU."""

import pytest

from test_operators_host import library


@pytest.mark.parametrize("columns", [(1 << 24) + 32, 1 << 30])
def test_more_columns_than_the_products_take_are_refused(columns):
    lib, null = library(), None
    assert lib.nanoep_experts_linear(64, 128, 64, 1, 64, 64, null, null, 1, 1, 128, columns, 64, null) == 1
    assert lib.nanoep_experts_gated(64, 128, 64, 1, 64, 64, null, null, 1, 1, 128, columns, 64, 64, 1 << 40, null) == 1
