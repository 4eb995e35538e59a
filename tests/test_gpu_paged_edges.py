"""The paged-cache operators on the GPU at the edges of what their callers may pass."""
import numpy as np
import pytest

from test_gpu_paged import TYPES, attend, check_attention, make
from test_gpu_paged import torch as torch  # the fixture

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- windows
@pytest.mark.parametrize("t,kv", TYPES)
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 64, 2**30])
@pytest.mark.parametrize("new,total", [([4, 1], [1, 30]), ([3, 2], [1, 0]), ([100], [60]), ([140], [3]), ([1, 90, 5], [9, 40, 5])])
def test_windows_wider_than_any_sequence(pkg, torch, t, kv, window, new, total):
    """No limit, given as a large window: as window 0, also with more new rows than positions."""
    rng = np.random.default_rng(sum(new) + sum(total))
    b, q, pages, pool = make(torch, rng, t, kv, new, total, 16, "slot", 4, 2, 64)
    got, gl, st = attend(pkg, torch, b, q, pool, t, window=window)
    assert st == 0
    check_attention(b, got, gl, q, pages, t, kv, 0.125, 0)
