"""Flat rows with one or a few logits far below the rest (a mask of -1e4 or -infinity). Bins spread down to these would put more
tokens into those of the draw and of top-p's border than the list of collected ones takes (4096), with no two of them equal, and
the row would be searched by one workgroup. The reference and its tolerance are test_sample_gpu's."""
import math

import numpy as np
import pytest
import torch

from soinfer import _C, ops
from test_sample_gpu import check

pytestmark = pytest.mark.gpu


LISTED = 8 * 1024 + 4 * 1024  # where a row's workspace says how many tokens were collected, behind 1024 sums and counts


def spread_to_the_lowest(l, u, T, p):
    """Tokens in the bins of the drawn token and of top-p's border, with bins of equal width down to the lowest logit."""
    z = np.sort((l.max() - l.astype(np.float64)) / T)
    bins = np.minimum(z * 1024 / min(z[-1], 45 * math.log(2)), 1023).astype(int)
    cum = np.cumsum(np.exp(-z))
    kept = cum[-1]
    at = set()
    if p < 1:
        i = min(int(np.searchsorted(cum, p * kept)), len(z) - 1)
        at.add(bins[i])
        kept = cum[i]
    at.add(bins[min(int(np.searchsorted(cum, u * kept, side="right")), len(z) - 1)])
    return sum(int((bins == b).sum()) for b in at)


@pytest.mark.parametrize("V,spread", [(151936, 0.35), (262144, 0.55), (524288, 0.75)])
@pytest.mark.parametrize("p", [1.0, 0.3, 0.9])
@pytest.mark.parametrize("low,how_many", [(-1e4, 1), (-1e4, 30), (-300.0, 1), (-math.inf, 2)])
def test_a_flat_row_with_logits_far_below(cuda, V, spread, p, low, how_many):
    g = torch.Generator(device=cuda).manual_seed(V + how_many)
    clean = torch.randn(4, V, generator=g, device=cuda) * spread
    x = clean.clone()
    x[:, torch.randint(0, V, (how_many,), generator=g, device=cuda)] = low
    u = torch.tensor([0.3, 0.5, 0.62, 0.97], device=cuda)
    if low > -math.inf:
        most = max(spread_to_the_lowest(x[b].cpu().numpy(), u[b].item(), 1.0, p) for b in range(4))
        assert most > 4096, most  # (the rows are what this test is for)
    ws = torch.empty(_C.sample_tokens_workspace_bytes(1, V), dtype=torch.uint8, device=cuda)
    for b in range(4):
        listed = []
        for row in (clean, x):
            ops.sample_tokens(row[b:b + 1], u[b:b + 1], 1.0, 0, p, workspace=ws)
            listed.append(ws[LISTED:LISTED + 4].view(torch.int32).item())
        # (as many as without the masks, but for wider bins of a lower median and one more of them; eight times as many or more
        # with bins down to the lowest)
        assert 0 < listed[1] <= 2 * listed[0], listed
    check(x, u, 1.0, 0, p, 0.0, close_allowed=1)
    check(x, u, 1.0, 4000, p, 0.0, close_allowed=1)
    check(x, u, torch.tensor([1.0, 0.7, 2.0, 1.0], device=cuda), 0, p, 1e-3, close_allowed=1)


@pytest.mark.parametrize("V", [600, 9000, 40000, 151936])
def test_rows_of_several_levels(cuda, V):
    """Blocks of the vocabulary at levels of their own: constant ones, masked ones, most of the row masked, few logits left."""
    g = torch.Generator(device=cuda).manual_seed(V)
    x = torch.randn(8, V, generator=g, device=cuda) * 0.5
    x[1, V // 2:] -= 4.0
    x[2, : 2 * V // 3] -= 15.0
    x[3, V // 3:] = -1e4
    x[4, V // 10:] = -math.inf
    x[5, : V // 2] = 3.0                # above most others, and equal
    x[6, 5:] = -20.0
    x[7, ::2] = -math.inf
    x[7, 1::4] -= 30.0
    u = torch.tensor([0.1, 0.9, 0.999, 0.5, 0.5, 0.97, 0.999, 0.5], device=cuda)
    for s in ((1.0, 0, 1.0, 0.0), (2.0, 0, 0.9, 0.0), (0.5, 3000, 0.99, 0.01), (1.0, 40, 0.95, 0.0), (30.0, 0, 0.5, 0.2)):
        check(x, u, *s, close_allowed=1)
        check(x.half(), u, *s, close_allowed=1)
