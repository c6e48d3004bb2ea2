"""The operators over a model's columns at the edges of what they accept: sums that leave fp32 on either side, log-sums that
hold few digits, empty matrices, operands that lie between one another, and calls from two threads.

Tolerances are those of test_gpu_columns.py: 2^-24 per fp32 operation, half a step of the output's type for its rounding.
"""
import ctypes as C
import threading

import numpy as np
import pytest

import columns_ref as ref
from bidmat_amd.device import DeviceArray
from bidmat_amd.mats import DDS, GMat, GSMat, Mat
from columns_ref import EPS24, HALF_STEP, TINY, TYPES, decode, encode, np_type
from test_gpu_columns import NORM_DEPTH, Columns, dev, empty, norm_case, ok, ptr, teacher, within

pytestmark = pytest.mark.gpu
F = np.float32
MOST = {0: 3.4028234663852886e38, 1: 65504.0, 2: 3.3895313892515355e38}      # largest finite value of a type


# ---------------------------------------------------------------- normalisation: sums outside fp32
HEIGHTS = [1, 2, 40, 300, 1001, 4096, 9000, 32768]


@pytest.mark.parametrize("n", HEIGHTS)
@pytest.mark.parametrize("t", [0, 2])
def test_rmsnorm_of_the_largest_values(hip, n, t):
    """Squares whose sum leaves fp32 by up to the largest finite values in every row, and eps that counts beside them."""
    rng = np.random.default_rng(n + t)
    x = rng.standard_normal((6, n))
    x[0] = 1e37
    x[1] = MOST[t] * np.where(np.arange(n) % 2, -1, 1)
    x[2, :2] = MOST[t]
    x[3] = 1e35
    x[4] *= 1e19
    for eps in (0.0, 1e-5, 1e36, 3.4e38):
        for group in (0, 32):
            norm_case(hip, rng, n, 6, t, False, True, True, group, x=x, eps=eps)
