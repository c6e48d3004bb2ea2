"""Sizes at which the kernels' 32-bit indices would leave the operands: refused before any work on a device (1 is
hipErrorInvalidValue). Addresses are made up and never read."""
import pytest

from test_columns_refusals import q8


@pytest.mark.parametrize("k", [2 ** 30 + 1, 2 ** 31 - 1])
def test_dsmult_q8_rows(k):
    assert q8(k=k, ldq=k, ncols=1, Q=1 << 40, C=1 << 44) == 1
