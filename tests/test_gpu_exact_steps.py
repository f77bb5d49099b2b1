"""Whole exact caches on the GPU: results do not depend on how rows and tokens are dealt to workgroups. Tolerances are those of
``test_gpu_exact_cache``."""
import math

import pytest
import torch

from test_gpu_exact_cache import Cache, attend, check, query

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ec(pkg):
    return pkg.exact_cache


@pytest.mark.parametrize('bad', [math.nan, math.inf])
@pytest.mark.parametrize('shares', [None, 0, 1, 8, 1024])
def test_rows_of_no_weight_whose_values_are_not_finite(ec, shares, bad):
    """A stretch of rows with scores of -inf: 0 * NaN and 0 * inf are NaN where the token has other rows, in a share of their own
    (with 1024 shares of 128 rows) as in one with others; a token that has nothing else gives 0 and -inf."""
    n = [1000, 1000, 300]
    c = Cache(80, n, 2, 128, 16)
    q = query(81, 3, 4, 128)
    q[:, :, 0] = 1
    for r, rows, kv_head in ((0, range(256, 384), 1), (1, range(0, 16), 0), (2, range(300), 1)):
        for j in rows:
            page, at = int(c.table[r, j // 16]), j % 16
            c.cache[page, :, at, 0] = -math.inf
            c.cache[page, kv_head, at, 128:] = bad
    o, lse = attend(ec, q, c, n, shares=shares)
    assert torch.isnan(o[0, 2:]).all() and torch.isnan(o[1, :2]).all()
    assert torch.isfinite(o[0, :2]).all() and torch.isfinite(o[1, 2:]).all() and torch.isfinite(lse[:, :2]).all()
    assert (o[2] == 0).all() and torch.isneginf(lse[:, 2]).all()
    c.rows[0], c.rows[1] = torch.cat((c.rows[0][:256], c.rows[0][384:])), c.rows[1][16:]
    for t, heads in ((0, slice(0, 2)), (1, slice(2, 4))):
        part = Cache.__new__(Cache)
        part.h, part.rows = 1, [c.rows[t][:, heads.start // 2:heads.stop // 2]]
        check(o[t:t + 1, heads].contiguous(), lse[heads, t:t + 1], q[t:t + 1, heads], part, [0], [c.rows[t].shape[0]], 128 ** -0.5)
