"""Decode attention where one token's V stands far above its neighbours', whichever of the eight tokens whose scales a lane
holds it is: the base of the weights follows it, and no product of weight and scale leaves binary16. Tolerance as in
test_kv4_range_gpu."""
import math

import numpy as np
import pytest
import torch

import kv4_ref as R
from test_kv4_range_gpu import cache_of, expect

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,gs,page", [(64, 32, 64), (128, 128, 16), (256, 64, 64)])
@pytest.mark.parametrize("at", range(8))
def test_one_large_v(cuda, hd, gs, page, at):
    import soinfer.ops as ops

    n, NQ, NKV = 200, 2, 1
    rng = np.random.RandomState(at)
    q, k = rng.randn(NQ, hd).astype(np.float16), rng.randn(n, NKV, hd).astype(np.float16)
    v = rng.randn(n, NKV, hd) * 2.0 ** -6
    for t in (at, 72 + at):
        k[t] = q.mean(0) * 0.5  # seen well
        v[t] *= 2.0 ** 14
    c, table, lt, held = cache_of(cuda, [k], [v.astype(np.float16)], page, gs, at)
    qd = torch.from_numpy(q).to(cuda)[None]
    got = ops.kv4_decode_attention(qd, *c, table, lt)
    ref, bound = expect(qd[0].double(), *held[0], 1 / math.sqrt(hd))
    R.assert_within(got[0], ref, bound, f"token {at} of 8")
