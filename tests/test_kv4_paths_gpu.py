"""Decode attention and prompt attention where one pass over the batch or the splits is not enough: more than 64 sequences,
more than 32 and 64 splits of a context, more than 32 splits of a prompt's keys."""
import math

import numpy as np
import pytest
import torch

import kv4_ref as R
from test_kv4_gpu import append_problem, append_ref, check_attention, queries, run_append, same_cache
from test_kv4_range_gpu import cache_of

pytestmark = pytest.mark.gpu


def context(dev, lens, NKV, hd, gs, page, seed):
    rng = np.random.RandomState(seed)
    ks, vs = ([rng.randn(max(1, n), NKV, hd).astype(np.float16) for n in lens] for _ in range(2))
    c, table, _, held = cache_of(dev, ks, vs, page, gs, seed)
    return c, table, torch.tensor(lens, dtype=torch.int32, device=dev), [[x[:n] for x in h] for h, n in zip(held, lens)]


@pytest.mark.parametrize("B", [64, 65, 130, 200])
@pytest.mark.parametrize("NQ,NKV,hd,gs,page", [(4, 2, 64, 32, 16), (4, 1, 128, 64, 64), (2, 1, 256, 128, 64)])
def test_many_sequences(cuda, B, NQ, NKV, hd, gs, page):
    """Empty, short and split contexts, first and last in their 64 among them."""
    import soinfer.ops as ops

    lens = np.random.RandomState(B).randint(0, 200, B)
    lens[[x for x in (0, 63, 64, 127) if x < B]] = 0
    for at, n in ((1, 1700), (62, 900), (66, 257), (128, 64), (B - 1, 2100)):
        lens[at % B] = n
    c, table, lt, held = context(cuda, lens.tolist(), NKV, hd, gs, page, B)
    q = queries(cuda, B, NQ, hd, B)
    got = ops.kv4_decode_attention(q, *c, table, lt, max_len=2100)
    check_attention(got, q, held, f"B {B}")
    assert (got[torch.from_numpy(lens == 0).to(cuda)] == 0).all()
    assert torch.equal(got, ops.kv4_decode_attention(q, *c, table, lt, max_len=2100))


@pytest.mark.parametrize("L", [8193, 16384, 20000])
@pytest.mark.parametrize("NQ,NKV,hd,gs,page", [(2, 1, 64, 64, 64), (3, 1, 128, 32, 16), (17, 1, 256, 64, 256)])
def test_more_splits_than_a_wave_has_lanes(cuda, L, NQ, NKV, hd, gs, page):
    """Splits of 256 tokens: 33, 64 and 79 of them, and a short neighbour."""
    import soinfer.ops as ops

    c, table, lt, held = context(cuda, [L, 70], NKV, hd, gs, page, L)
    q = queries(cuda, 2, NQ, hd, L)
    got = ops.kv4_decode_attention(q, *c, table, lt, max_len=L)
    check_attention(got, q, held, f"L {L}")
    alone = ops.kv4_decode_attention(q[:1].contiguous(), *c, table[:1].contiguous(), lt[:1].contiguous(), max_len=L)
    check_attention(alone, q, held[:1], f"L {L} alone")


@pytest.mark.parametrize("hd,keys", [(64, 17000), (128, 4300), (128, 9000), (200, 17000)])
@pytest.mark.parametrize("nq", [1, 33])
def test_prompt_keys_in_many_splits(cuda, hd, keys, nq):
    import soinfer._C as _C
    import soinfer.ops as ops

    NQ, NKV = 2, 1
    g = torch.Generator(device=cuda).manual_seed(keys + nq)
    q, k, v = (torch.randn((n, h, hd), generator=g, device=cuda).half() for n, h in ((nq, NQ), (keys, NKV), (keys, NKV)))
    splits = _C.prompt_attention_workspace_bytes(nq, keys, NQ, hd) // (nq * NQ * (hd + 2) * 4)
    assert splits > 32
    at = lambda n: torch.tensor([0, n], dtype=torch.int32, device=cuda)  # noqa: E731
    got = ops.prompt_attention(q, k, v, at(nq), at(keys), nq)
    last = torch.arange(nq, device=cuda) + keys - nq
    ref, bound = R.attention(q.double(), k.double(), v.double(), last, 1 / math.sqrt(hd))
    R.assert_within(got, ref, bound, f"{splits} splits")


def test_append_to_a_thousand_sequences(cuda):
    """Zero to four new tokens each: most are found by counting the sequences' ends."""
    NQ, NKV, hd, gs, page, B = 2, 1, 64, 32, 16, 1000
    rng = np.random.RandomState(1)
    p = append_problem(cuda, rng.randint(0, 20, B).tolist(), rng.randint(0, 5, B).tolist(), NQ, NKV, hd, gs, page, True, 1)
    ref, q, _ = append_ref(p, NQ, NKV, hd, gs, page, 1e-6)
    c, qo, _ = run_append(cuda, p, NQ, NKV, hd, gs, page)
    same_cache(c, ref)
    R.same(qo, R.half(q), "q")
