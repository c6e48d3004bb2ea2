"""Sizes at which the kernels' 32-bit indices would leave the operands: refused before any work on a device (1 is
hipErrorInvalidValue). Addresses are made up and never read."""
import pytest

from test_columns_refusals import distill, distill_grad, q8


@pytest.mark.parametrize("k", [2 ** 30 + 1, 2 ** 31 - 1])
def test_dsmult_q8_rows(k):
    assert q8(k=k, ldq=k, ncols=1, Q=1 << 40, C=1 << 44) == 1


@pytest.mark.parametrize("nnz", [2 ** 31 - 1024, 2 ** 31 - 1])
def test_distill_stored_values(nnz):
    assert distill(nnz=nnz, T=1 << 40, ir=1 << 44, Z=1 << 46, dZ=1 << 47, jc=1 << 48) == 1
    assert distill_grad(nnz=nnz, T=1 << 40, ir=1 << 44, Z=1 << 46, dZ=1 << 47, jc=1 << 48) == 1
