"""Attention of sequences that share their first pages: how far the weights are rounded, and V of any size.

A product of weight and V scale is kept as two binary16 numbers, so it is off by 2^-22 of itself (u^2), or by 2^-25 where that is
more. The largest one that a unit of work has met is 2^12 or more when its V scale is taken as the next power of two, so 2^11 or
more as it is: 2^-36 of it a token, times a code of up to 7, which is 2^-36 max|v|. Else as kv4_ref: the output's rounding, a
score's d = (hd + 8) e sum |q k| scale + 2^-19 (arguments of the exponential below 64), and sums of n terms in binary32, those of
the weights too.
"""
import math

import numpy as np
import pytest
import torch

import kv4_ref as R
from soinfer import ops
from test_kv4_range_gpu import cache_of

pytestmark = pytest.mark.gpu

SHAPES = [(64, 32, 16), (64, 64, 64), (128, 32, 64), (128, 64, 32), (128, 128, 64), (256, 32, 16), (256, 64, 64), (256, 128, 128)]
COLUMNS = [(2, 2), (12, 4), (20, 4)]  # sequences, query heads of a KV head: one, two and four tiles of 32 columns side by side


def grouped(dev, prefix, tails, page, gs, seed, copies=1):
    """One group of sequences: prefix (k, v) of whole pages, the (k, v) behind it of each; `copies` sequences of each tail, whose
    pages are the same but not named as shared. (cache, the operator's tables, and what each sequence holds, binary64)."""
    n = len(prefix[0])
    assert n % page == 0
    c, rows, lens, held = cache_of(dev, [prefix[0]] + [k for k, _ in tails], [prefix[1]] + [v for _, v in tails], page, gs, seed)
    B = len(tails) * copies
    table = torch.cat([rows[:1, :n // page].expand(B, -1), rows[1:].repeat(copies, 1)], 1).contiguous()
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    held = [[torch.cat([held[0][i], own[i]]) for i in range(2)] for own in held[1:]] * copies
    return c, (table, lens[1:].repeat(copies) + n, i32([0, B]), i32([n] * B)), held


def expect(q, k, v, scale):
    """(out, bound) of one query [NQ, hd] over k, v [n, NKV, hd], 64 bits."""
    NQ, hd = q.shape
    n, NKV = k.shape[:2]
    kh, vh = (x.repeat_interleave(NQ // NKV, 1).transpose(0, 1) for x in (k, v))  # [NQ, n, hd]
    z = (kh * q[:, None]).sum(-1) * scale
    d = ((kh * q[:, None]).abs().sum(-1).amax(-1) * scale * (hd + 8) * R.E + 2.0 ** -19)[:, None]
    p = torch.exp(z - z.amax(-1, keepdim=True))[..., None]
    tot = p.sum(1)
    out, A = (p * vh).sum(1) / tot, (p * vh.abs()).sum(1) / tot
    most = vh.abs().amax((1, 2))[:, None]
    return out, R.U * out.abs() + R.TINY + (R.U * R.U + 2 * d + 3 * n * R.E) * A + n * 2.0 ** -36 * most / tot


def check(c, tables, held, q, label, pick=None):
    got = ops.kv4_shared_attention(q, *c, *tables)
    assert torch.isfinite(got).all(), label
    for b in range(len(held)) if pick is None else pick:
        ref, bound = expect(q[b].double(), *held[b], 1 / math.sqrt(q.shape[2]))
        R.assert_within(got[b], ref, bound, f"{label}, sequence {b}")


@pytest.mark.parametrize("hd,gs,page", SHAPES)
@pytest.mark.parametrize("B,rep", COLUMNS)
def test_a_weight_is_not_rounded_to_binary16(cuda, hd, gs, page, B, rep):
    """One token has a V, so an output is one weight times one value: a weight rounded to 2^-11 would leave the bound of the
    output's own rounding. Scores are small and so are their errors."""
    rng = np.random.RandomState(B + hd)
    rows = lambda n: (rng.randn(n, 1, hd).astype(np.float16), np.zeros((n, 1, hd), np.float16))  # noqa: E731
    q = torch.from_numpy((0.1 * rng.randn(B, rep, hd)).astype(np.float16)).to(cuda)
    prefix, tails = rows(128), [rows(60 + b) for b in range(B)]
    for at in (5, 100, None):  # of the shared tokens, or of each sequence's own
        prefix[1][:] = 0
        for _, v in tails:
            v[:] = 0
            if at is None:
                v[rng.randint(len(v))] = rng.randn(hd) * 8
        if at is not None:
            prefix[1][at] = rng.randn(hd) * 8
        check(*grouped(cuda, prefix, tails, page, gs, 1), q, f"V of token {at}")


@pytest.mark.parametrize("hd,gs,page", SHAPES)
@pytest.mark.parametrize("B,rep", COLUMNS)
def test_small_scores(cuda, hd, gs, page, B, rep):
    rng = np.random.RandomState(B + hd + 1)
    rows = lambda n: tuple(rng.randn(n, 2, hd).astype(np.float16) for _ in range(2))  # noqa: E731
    q = torch.from_numpy((0.1 * rng.randn(B, 2 * rep, hd)).astype(np.float16)).to(cuda)
    check(*grouped(cuda, rows(256), [rows(1 + 17 * b) for b in range(B)], page, gs, 2), q, "small scores")


@pytest.mark.parametrize("hd,gs,page", SHAPES[::2] + SHAPES[-1:])
@pytest.mark.parametrize("B,rep", COLUMNS)
@pytest.mark.parametrize("at", range(16))
def test_one_large_v(cuda, hd, gs, page, B, rep, at):
    """One token's V stands far above its neighbours' in one scale group, at each place of 16 tokens, in the first and in a later
    stage of the shared tokens, and behind them: the base of the weights follows it, and no product leaves binary16."""
    rng = np.random.RandomState(at)
    q = rng.randn(B, rep, hd).astype(np.float16)
    groups = hd // gs
    dims = slice(at % groups * gs, (at % groups + 1) * gs)
    pick = (0, B - 1)

    def rows(n, large=None):
        k, v = rng.randn(n, 1, hd), rng.randn(n, 1, hd) * 2.0 ** -6
        if large is not None:
            k[large] = q.mean((0, 1)) * 0.5  # seen well
            v[large, :, dims] *= 2.0 ** 14
        return k.astype(np.float16), v.astype(np.float16)

    qd = torch.from_numpy(q).to(cuda)
    for label, n, where in (("first stage", 256, at + 16 * (at % 4)), ("later stage", 256, 128 + at + 16 * ((at + 1) % 4)),
                            ("own tokens", 128, None)):
        tails = [rows(80, 16 * ((at + b) % 5) + at if where is None else None) for b in range(B)]
        check(*grouped(cuda, rows(n, where), tails, page, gs, at), qd, f"{label}, place {at}", pick)


@pytest.mark.parametrize("hd,gs,page", SHAPES)
@pytest.mark.parametrize("B", [10, 24, 40])
@pytest.mark.parametrize("strong", [[], [130], [1400], [5, 700, 1533, 2100]])
def test_sizes_that_change(cuda, hd, gs, page, B, strong):
    """V of another size every 150 tokens, up and down, with strong keys here and there whose own V is 0: units of several stages
    (8 KV heads share the workgroups), shared tokens and others."""
    rng = np.random.RandomState(B + len(strong))
    n, NKV, shared = 2236, 8, 1536
    u = rng.choice([-1.0, 1.0], hd)
    q = torch.from_numpy((u + 0.05 * rng.randn(B, 2 * NKV, hd)).astype(np.float16)).to(cuda)
    sizes = (2.0 ** np.array([-12, -3, -9, 0, -6, 4, -12, 8, -2, -12]))[np.arange(n) // 150 % 10]

    def rows(lo, hi):
        k, v = rng.randn(hi - lo, NKV, hd), (rng.randn(hi - lo, NKV, hd) + 0.5) * sizes[lo:hi, None, None]
        for t in strong:
            if lo <= t < hi:
                k[t - lo] = u * 12 / math.sqrt(hd)
                v[t - lo] = 0
        return k.astype(np.float16), v.astype(np.float16)

    check(*grouped(cuda, rows(0, shared), [rows(shared, n)], page, gs, 3, B), q, f"strong {strong}", (0, 3, B - 1))


@pytest.mark.parametrize("strong", [[5], [1500], list(range(7, 3001, 64))])
@pytest.mark.parametrize("first,then", [(2.0 ** -10, 16.0), (16.0, 2.0 ** -10), (2.0 ** -14, 9000.0 * 7)])
def test_sizes_up_to_the_largest_number(cuda, first, then, strong):
    rng = np.random.RandomState(4)
    n, hd, shared, B = 3001, 64, 1024, 30
    u = rng.choice([-1.0, 1.0], hd)
    k, v = rng.randn(n, 1, hd), np.clip(rng.randn(n, 1, hd) + 0.5, -1, 1)
    k[strong], v[strong] = u * 12 / math.sqrt(hd), 0
    v[:1500] *= first
    v[1500:] *= then
    k, v = k.astype(np.float16), v.astype(np.float16)
    q = torch.from_numpy((u + 0.05 * rng.randn(B, 2, hd)).astype(np.float16)).to(cuda)
    check(*grouped(cuda, (k[:shared], v[:shared]), [(k[shared:], v[shared:])], 64, 32, 5, B), q, f"{first} {then}", (0, B - 1))
