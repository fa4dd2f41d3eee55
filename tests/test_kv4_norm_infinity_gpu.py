"""An infinity or NaN in a head that is normed before its rotation: what the formula makes of it, and no more."""
import numpy as np
import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,gs", [(64, 32), (128, 32), (128, 64), (256, 32), (256, 64)])
@pytest.mark.parametrize("at", [3, -1])
def test_an_infinity_before_the_norm(cuda, hd, gs, at):
    """The mean square is infinite: finite elements become 0 and the infinity NaN, which the rotation carries to the other
    half's element of its pair. Two groups of the cached k are then NaN (or the one that holds both), the others 0."""
    import soinfer.ops as ops

    NQ, NKV, page, rng = 2, 1, 16, np.random.RandomState(hd)
    up = lambda x: torch.from_numpy(x).to(cuda)  # noqa: E731
    for bad in (np.inf, -np.inf, np.nan):
        qkv = rng.randn(3, NQ + 2 * NKV, hd).astype(np.float16)
        qkv[1, :NQ + NKV, at] = bad
        w = [(1 + 0.2 * rng.randn(hd)).astype(np.float16) for _ in range(2)]
        cos, sin = R.rope_tables(3, hd)
        c = R.Cache(1, NKV, page, hd, gs).tensors(cuda)
        t = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
        k_out = torch.empty((3, NKV, hd), dtype=torch.float16, device=cuda)
        q = ops.kv4_append(up(qkv.reshape(3, -1)), up(w[0]), up(w[1]), up(cos), up(sin), *c, t(0)[None], t(3), t(0, 3), NQ,
                           k_out=k_out)
        for r in range(3):
            with np.errstate(invalid="ignore"):
                for got, x, weight in ((q[r], qkv[r, :NQ], w[0]), (k_out[r], qkv[r, NQ:NQ + NKV], w[1])):
                    want = R.half(R.norm_rope(x, weight, 1e-6, cos[r], sin[r]))
                    assert np.array_equal(got.cpu().numpy(), want, equal_nan=True), f"row {r} of {bad}"
        k, v = ops.kv4_read(*c, t(0)[None], t(3), t(0, 3), 3)
        pair = {(at % hd) // gs, ((at % hd) + hd // 2) % hd // gs}
        for g in range(hd // gs):
            part = k[1, 0, g * gs:(g + 1) * gs]
            assert torch.isnan(part).all() if g in pair or np.isnan(bad) else (part == 0).all()
        assert torch.isfinite(k[[0, 2]]).all() and torch.isfinite(v).all()
