"""Prompt attention where most keys' weights are far below the largest one.

The strong key's own V is 0, so the output is made of the others. Tolerance (u, e as in kv4_ref): the weights are rounded
once to binary16, and the sum takes them rounded: u (A + |ref|); below binary16's normal range they are rounded to within
2^-25, where the largest weight of a row is at least 2^7: 2^-32 of it a key, in the products and in the sum.
"""
import math

import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu


def expect(q, k, v, last, scale):
    n, NQ, hd = q.shape
    m, NKV = k.shape[:2]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    seen = torch.arange(m, device=q.device)[None] <= last[:, None]
    far = seen.sum(-1, keepdim=True).double()
    for h in range(NQ):
        kh, vh = k[:, h * NKV // NQ], v[:, h * NKV // NQ]
        z = torch.where(seen, q[:, h] @ kh.T * scale, -torch.inf)
        d = torch.where(seen, q[:, h].abs() @ kh.abs().T, 0).amax(-1, keepdim=True) * scale * (hd + 8) * R.E + 2.0 ** -19
        p = torch.exp(z - z.amax(-1, keepdim=True))
        tot = p.sum(-1, keepdim=True)
        o, A = p @ vh / tot, p @ vh.abs() / tot
        out[:, h] = o
        bound[:, h] = R.U * o.abs() + R.TINY + R.U * (A + o.abs()) + (2 * d + 2 * far * R.E) * A + \
            2 * far * vh.abs().amax() * 2.0 ** -32 / tot
    return out, bound


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("NQ,NKV,nq,nk", [(4, 2, 40, 8200), (16, 4, 2500, 2500)])
@pytest.mark.parametrize("gap", [12, 17])
def test_weights_far_below_the_largest(cuda, hd, NQ, NKV, nq, nk, gap):
    """The strong key is the first one, so every query sees it; few queries (their keys split) and many."""
    import soinfer.ops as ops

    g = torch.Generator(device=cuda).manual_seed(hd + gap)
    rn = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    u = torch.sign(rn(hd))
    q = (u + 0.05 * rn(nq, NQ, hd)).half()
    k, v = 0.5 * rn(nk, NKV, hd), 1 + 0.1 * rn(nk, NKV, hd)
    k[0], v[0] = u * gap / math.sqrt(hd), 0
    k, v = k.half(), v.half()
    at = lambda n: torch.tensor([0, n], dtype=torch.int32, device=cuda)  # noqa: E731
    got = ops.prompt_attention(q, k, v, at(nq), at(nk), nq)
    last = torch.arange(nq, device=cuda) + nk - nq
    ref, bound = expect(q.double(), k.double(), v.double(), last, 1 / math.sqrt(hd))
    R.assert_within(got, ref, bound, f"gap {gap}")
