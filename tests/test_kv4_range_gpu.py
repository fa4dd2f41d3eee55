"""Decode attention over V of any size, with a key that stands far above the rest: the products of weight and V scale stay
within what their binary16 operand holds.

A strong key's own V is 0, as an attention sink's is, so the output is made of weights far below the largest. Tolerance (u, e
as in kv4_ref): a product of weight and scale is rounded once, u A, or to within 2^-25 where it is below binary16's normal
range; the largest product of a wave is kept in [2^14, 2^15), so that is 2^-39 of the largest weight times the largest scale
a token, and a code is at most 7 and max|v| is 7 scales. The exponent's argument is below 64, so it is rounded to within 2^-19.
"""
import math

import numpy as np
import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu


def k_bytes(q):
    """codes [P, NKV, page, hd] -> k_pages."""
    w = q.shape[-1] // 32
    o = (q & 15).astype(np.uint32).reshape(*q.shape[:-1], -1, 8)
    words = sum(o[..., R.AWQ[n]] << np.uint32(4 * n) for n in range(8))
    order = [4 * i + g for g in range(4) for i in range(w)]
    return np.ascontiguousarray(words[..., order]).view(np.uint8)


def v_bytes(q):
    """codes [P, NKV, page, hd] -> v_pages."""
    P, NKV, page, hd = q.shape
    o = (q & 15).astype(np.uint16).reshape(P, NKV, page // 4, 4, hd // 64, 4, 16)  # .., token, u, nibble, m
    units = sum(o[..., n, :] << np.uint16(4 * n) for n in range(4)).transpose(0, 1, 2, 5, 4, 3)
    return np.ascontiguousarray(units).reshape(P, NKV, -1).view(np.uint8).reshape(P, NKV, page, hd // 2)


def cache_of(dev, ks, vs, page, gs, seed):
    """Sequences' K and V [n, NKV, hd] fp16 -> (pages in any order, block table, lengths, held values per sequence)."""
    NKV, hd = ks[0].shape[1:]
    lens = [len(k) for k in ks]
    counts = [-(-n // page) for n in lens]
    P = sum(counts) + 1
    order = np.random.RandomState(seed).permutation(P)
    table = np.full((len(lens), max(1, *counts)), -1, np.int32)
    raw, scale, held = np.zeros((2, P, NKV, page, hd), np.int8), np.full((2, P, NKV, hd // gs, page), np.nan, np.float16), []
    at = 0
    for b, n in enumerate(lens):
        pg = order[at:at + counts[b]]
        table[b, :counts[b]], at = pg, at + counts[b]
        t = np.arange(n)
        h = []
        for x, src in enumerate((ks[b], vs[b])):
            q, s = R.quantize(src, gs)
            raw[x, pg[t // page], :, t % page] = q
            scale[x, pg[t // page], :, :, t % page] = s
            h.append(torch.from_numpy(R.values(q, s)).to(dev))
        held.append(h)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    c = (up(k_bytes(raw[0])), up(scale[0]), up(v_bytes(raw[1])), up(scale[1]))
    return c, up(table), torch.tensor(lens, dtype=torch.int32, device=dev), held


def strong_key(dev, n, NQ, NKV, hd, gap, size, strong, seed):
    """q [NQ, hd], K and V [n, NKV, hd]: scores of deviation 1, those of the tokens `strong` `gap` above their mean, with V 0
    there and of deviation `size` around half of it elsewhere."""
    rng = np.random.RandomState(seed)
    u = rng.choice([-1.0, 1.0], hd)
    q = u + 0.05 * rng.randn(NQ, hd)
    k = rng.randn(n, NKV, hd)
    v = (rng.randn(n, NKV, hd) + 0.5) * size
    k[strong] = u * gap / math.sqrt(hd)
    v[strong] = 0
    return q.astype(np.float16), k.astype(np.float16), v.astype(np.float16)


def expect(q, k, v, scale):
    """(out, bound) of one query [NQ, hd] over k, v [n, NKV, hd], 64 bits."""
    NQ, hd = q.shape
    n, NKV = k.shape[:2]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(NQ):
        kh, vh = k[:, h * NKV // NQ], v[:, h * NKV // NQ]
        z = kh @ q[h] * scale
        d = (kh.abs() @ q[h].abs()).amax() * scale * (hd + 8) * R.E + 2.0 ** -19
        p = torch.exp(z - z.amax())
        tot = p.sum()
        A = p @ vh.abs() / tot
        out[h] = p @ vh / tot
        bound[h] = R.U * out[h].abs() + R.TINY + (R.U + 2 * d + 2 * n * R.E) * A + n * vh.abs().amax() * 2.0 ** -39 / tot
    return out, bound


def test_packed_like_the_reference():
    rng = np.random.RandomState(0)
    for hd in (64, 128, 256):
        q = rng.randint(-7, 8, (1, 1, 16, hd)).astype(np.int8)
        c = R.Cache(1, 1, 16, hd, 32)
        for t in range(16):
            c.k[0, 0, t] = R.k_row_bytes(q[0, 0, t])
            units = c.v[0, 0].view(np.uint16).reshape(4, 16, hd // 64, 4)
            for (m, u), x in R.v_row_units(q[0, 0, t]).items():
                units[t // 4, m, u, t % 4] = x
        assert np.array_equal(c.k, k_bytes(q)) and np.array_equal(c.v, v_bytes(q))


@pytest.mark.parametrize("hd,gs,page", [(64, 32, 16), (128, 64, 64), (128, 128, 16), (256, 64, 64)])
@pytest.mark.parametrize("n", [200, 4100])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -6, 2.0 ** -10])
@pytest.mark.parametrize("gap", [10, 14])
def test_weights_far_below_the_largest(cuda, hd, gs, page, n, size, gap):
    import soinfer.ops as ops

    NQ, NKV = 4, 2
    q, k, v = strong_key(cuda, n, NQ, NKV, hd, gap, size, [n // 3], n + gap)
    c, table, lt, held = cache_of(cuda, [k], [v], page, gs, n)
    qd = torch.from_numpy(q).to(cuda)[None]
    got = ops.kv4_decode_attention(qd, *c, table, lt)
    ref, bound = expect(qd[0].double(), *held[0], 1 / math.sqrt(hd))
    R.assert_within(got[0], ref, bound, f"size {size} gap {gap}")


@pytest.mark.parametrize("first,then", [(2.0 ** -10, 16.0), (16.0, 2.0 ** -10), (2.0 ** -14, 9000.0 * 7)])
def test_sizes_that_change_along_the_context(cuda, first, then):
    """V grows or shrinks by many binades after its first tokens, up to scales near the largest number: the products follow,
    and do not leave binary16 at the top either. A strong key near the beginning, one near the end, one in every 64 tokens."""
    import soinfer.ops as ops

    n, NQ, NKV, hd = 3001, 2, 1, 64
    for strong in ([5], [2990], list(range(7, n, 64))):
        q, k, v = strong_key(cuda, n, NQ, NKV, hd, 12, 1.0, strong, 3)
        v = np.clip(v.astype(np.float64), -1, 1)
        v[:1500] *= first
        v[1500:] *= then
        c, table, lt, held = cache_of(cuda, [k], [v.astype(np.float16)], 64, 32, 4)
        qd = torch.from_numpy(q).to(cuda)[None]
        got = ops.kv4_decode_attention(qd, *c, table, lt)
        ref, bound = expect(qd[0].double(), *held[0], 1 / math.sqrt(hd))
        R.assert_within(got[0], ref, bound, f"{first} {then} {len(strong)}")


def test_values_that_are_not_finite(cuda):
    """A cached group with an infinity or NaN: in V it spoils its own dimensions for the heads that read it and no others, in K
    every dimension of these heads, and neither reaches the other sequence."""
    import soinfer.ops as ops

    n, NQ, NKV, hd, gs = [700, 130], 6, 2, 128, 32
    rng = np.random.RandomState(6)
    ks, vs = ([rng.randn(m, NKV, hd).astype(np.float16) for m in n] for _ in range(2))
    vs[0][350, 1, 32:64] = 0  # the group that is spoilt below
    q = torch.from_numpy(rng.randn(2, NQ, hd).astype(np.float16)).to(cuda)
    run = lambda: ops.kv4_decode_attention(q, *cache_of(cuda, ks, vs, 64, gs, 6)[0], *rest)  # noqa: E731
    rest = cache_of(cuda, ks, vs, 64, gs, 6)[1:3]
    want = run()
    for bad in (np.inf, -np.inf, np.nan):
        vs[0][350, 1, 40] = bad
        got = run()
        assert torch.isnan(got[0, 3:, 32:64]).all()
        got[0, 3:, 32:64] = want[0, 3:, 32:64]
        assert torch.equal(got, want)
        vs[0][350, 1, 40] = 0
        ks[0][350, 1, 40], was = bad, ks[0][350, 1, 40]
        got = run()
        assert torch.isnan(got[0, 3:]).all()
        got[0, 3:] = want[0, 3:]
        assert torch.equal(got, want)
        ks[0][350, 1, 40] = was


@pytest.mark.parametrize("NQ,hd,gs,page", [(2, 64, 32, 64), (2, 128, 128, 16), (17, 256, 32, 64), (2, 256, 64, 16)])
@pytest.mark.parametrize("strong", [[], [130], [1400], [5, 700, 1533, 2900]])
def test_sizes_that_change_within_a_wave(cuda, NQ, hd, gs, page, strong):
    """256 sequences of the same pages, so that a wave takes three blocks of 64 tokens and more, and V of another size every
    150 tokens: up and down, with strong keys (whose own V is 0) here and there."""
    import soinfer.ops as ops

    n, B = 3001, 256
    q, k, v = strong_key(cuda, n, NQ, 1, hd, 12, 1.0, strong, hd)
    sizes = 2.0 ** np.array([-12, -3, -9, 0, -6, 4, -12, 8, -2, -12])
    v = (v * sizes[np.arange(n) // 150 % 10][:, None, None]).astype(np.float16)
    c, table, lt, held = cache_of(cuda, [k], [v], page, gs, 7)
    qd = torch.from_numpy(q).to(cuda)
    got = ops.kv4_decode_attention(qd.expand(B, -1, -1).contiguous(), *c, table.expand(B, -1).contiguous(), lt.expand(B).contiguous())
    ref, bound = expect(qd.double(), *held[0], 1 / math.sqrt(hd))
    R.assert_within(got[0], ref, bound, f"strong {strong}")
    R.assert_within(got[-1], ref, bound, f"strong {strong}, last")
