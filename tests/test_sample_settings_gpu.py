"""Rows' settings outside their ranges: what cuts nothing, and what leaves the first tokens only."""
import math

import pytest
import torch

from soinfer import ops
from test_sample_gpu import check, rows

pytestmark = pytest.mark.gpu


def column(value, B, dev, dtype=torch.float32):
    return torch.full((B,), value, dtype=dtype, device=dev)


@pytest.mark.parametrize("V", [5, 4097, 60000])
@pytest.mark.parametrize("k", [0, 30, 5000])
def test_first_tokens(cuda, V, k):
    x, u = rows(cuda, 6, V, V + k)
    x[1] = 1.0                      # all of them the largest
    x[2, 3] = x[2, 1] = 30.0        # two of them
    first = torch.argmax(x.float(), 1).tolist()
    for p in (0.0, -0.0, -1e-40, -0.5, -3e38, -math.inf):  # one token stays
        assert ops.sample_tokens(x, u, 1.0, k, column(p, 6, cuda)).tolist() == first, p
    for m in (1.0, 1.5, math.inf):                         # the largest ones
        got = check(x, u, 1.0, k, 1.0, column(m, 6, cuda), close_allowed=1)
        assert all(x[b, t] == x[b].max() for b, t in enumerate(got))


@pytest.mark.parametrize("V", [5, 4097, 60000])
def test_settings_that_cut_nothing(cuda, V):
    x, u = rows(cuda, 6, V, V)
    want = ops.sample_tokens(x, u, 0.8).tolist()
    for p in (1.0, 1.5, math.inf, math.nan):
        assert ops.sample_tokens(x, u, 0.8, 0, column(p, 6, cuda)).tolist() == want, p
    for m in (0.0, -0.0, -1.0, -math.inf, math.nan):
        assert ops.sample_tokens(x, u, 0.8, 0, 1.0, column(m, 6, cuda)).tolist() == want, m
    for k in (0, -1, -2 ** 31, V, 2 ** 31 - 1):
        assert ops.sample_tokens(x, u, 0.8, column(k, 6, cuda, torch.int32)).tolist() == want, k
