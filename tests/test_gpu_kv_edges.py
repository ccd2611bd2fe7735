"""Attention over the paged Q4_0 cache where a call leaves the ordinary: rows
behind the table beside values that are NaN."""
import math

import numpy as np
import pytest
import torch

from catseye_b200 import _lib
from test_gpu_kv import LONG, TYPES, check_attention, fill, make, randn, runs_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean(gpu):
    gpu.cats_gpu_clear_device_error()
    yield
    torch.cuda.synchronize()
    gpu.cats_gpu_clear_device_error()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mul,hint", [(1, 128), (3, 128), (1, LONG), (3, LONG)])
def test_rows_past_the_table_beside_a_nan(dtype, mul, hint):
    """A run that goes on past its sequence's table, its last position inside
    holding NaN: the rows behind it are zeros, not what lies behind the table."""
    c = make([128, 64], 1, 64)
    fill(c, [128, 64])
    v = randn(1, 1, 64, seed=4)
    v[0, 0, 5] = math.nan
    c.append(1, randn(1, 1, 64, seed=5), v, runs_of([(0, 1, 0, 127)]), 1)
    q = randn(4, mul, 64, seed=6).to(dtype)
    out = torch.full_like(q, 3)
    c.attention(1, out, q, runs_of([(0, 4, 0, 126)]), 4, hint)
    torch.cuda.synchronize()
    check_attention(c, 1, q, out, [(0, 1, 0, 126)], mul)
    o = out.double().cpu().numpy()
    assert np.isnan(o[1, :, :32]).all() and np.isfinite(o[1, :, 32:]).all()
    assert (o[2:] == 0).all()
    assert _lib.load().cats_gpu_device_error() == 0x40
