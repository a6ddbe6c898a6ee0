"""The block-scaled 8-bit operators where values are not finite, buffers change hands and memory counts."""
import math

import pytest
import torch

from test_fp8_gpu import E4M3, E5M2, TYPES, check_held, matrix
from venom_b200 import capi, fp8

pytestmark = pytest.mark.gpu


# ---- values that are not finite ----

def rows_of_nan(x):
    x[140:144] = math.nan                      # four rows that one thread of each sixteen holds


def patch_of_nan(x):
    x[8:12, 16:24] = math.nan                  # all that one thread holds


def patch_beside_an_infinity(x):
    x[8:12, 16:24], x[13, 100] = math.nan, -math.inf


def tile_of_nan(x):
    x[128:256, :128] = math.nan


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("f8", [E4M3, E5M2])
@pytest.mark.parametrize("where", [rows_of_nan, patch_of_nan, patch_beside_an_infinity, tile_of_nan])
@pytest.mark.parametrize("square", [False, True])
def test_nan_side_by_side_leaves_the_other_values(dtype, f8, where, square):
    """The largest finite value of a tile lies in the eight rows that a warp holds together with the NaN."""
    x = matrix(260, 300, 3, TYPES[dtype], 0.5)
    x[14, 30], x[137, 250], x[139, 20] = 1000.0, -3000.0, 2000.0
    where(x)
    q, t = fp8.quantize(x, f8, square=square, both=True)
    check_held(q, x, f8, square)
    check_held(t, x.t(), f8, square)
