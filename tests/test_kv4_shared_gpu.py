"""Attention of sequences that share their first pages against 64-bit references over the values the cache holds.

Tolerance (u = 2^-11, e = 2^-24, as kv4_ref.attention): the output's rounding, one of each weight times V scale (u A), a score's
d = (hd + 8) e sum |q k| scale + 2^-21, and sums of n terms in binary32, those of the weights too. The base of the exponents
keeps the largest weight times the largest V scale that meets it at 2^12 or more, and a product below binary16's normal range is
rounded to within 2^-25 (codes up to 7 times that): n 2^-37 max|v| / sum p.
"""
import math

import numpy as np
import pytest
import torch

import kv4_ref as R
from soinfer import _C, ops
from test_kv4_range_gpu import k_bytes, v_bytes

pytestmark = pytest.mark.gpu


class Cache(tuple):
    """(k_pages, k_scale, v_pages, v_scale); held: the K and V that these stand for, binary64 [P, NKV, page, hd]."""


def scene(dev, groups, NKV, hd, gs, page, seed, std=1.0, spare=2):
    """groups: [(shared tokens, [own tokens of each sequence])]. Pages in any order; slots that no token has hold NaN scales.
    Returns (cache tensors, table, lens, cu, shared)."""
    rng = np.random.RandomState(seed)
    rows, lens, shared, cu, at = [], [], [], [0], 0
    for n_shared, tails in groups:
        assert n_shared % page == 0
        first = list(range(at, at + n_shared // page))
        at += len(first)
        for t in tails:
            n = -(-t // page)
            rows.append(first + list(range(at, at + n)))
            at += n
            lens.append(n_shared + t)
            shared.append(n_shared)
        cu.append(cu[-1] + len(tails))
    P = at + spare
    order = rng.permutation(P)
    table = np.full((len(rows), max(1, *map(len, rows))), -1, np.int32)
    q = rng.randint(-7, 8, (2, P, NKV, page, hd)).astype(np.int8)
    s = (rng.rand(2, P, NKV, hd // gs, page) * 0.25 * std + 0.02).astype(np.float16)
    used = np.zeros((P, page), bool)
    for b, r in enumerate(rows):
        table[b, :len(r)] = order[r]
        t = np.arange(lens[b])
        used[table[b][t // page], t % page] = True
    s[:, ~used.any(-1)] = np.nan
    s = np.where(used[None, :, None, None, :], s, np.float16(np.nan))
    up = lambda a, dt=None: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    c = Cache((up(k_bytes(q[0])), up(s[0]), up(v_bytes(q[1])), up(s[1])))
    c.held = [up(q[i]).double() * up(s[i]).double().transpose(2, 3).repeat_interleave(gs, 3) for i in range(2)]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    return c, up(table), i32(lens), i32(cu), i32(shared)


def reference(c, table, lens, q, scale):
    """(out, bound) in 64 bits, sequence by sequence."""
    outs, bounds = [], []
    for b, n in enumerate(lens.tolist()):
        qb = q[b].double()
        out, bound = torch.zeros_like(qb), torch.full_like(qb, R.TINY)
        if n:
            t = torch.arange(n, device=q.device)
            k, v = (x[table[b].long()[t // x.shape[2]], :, t % x.shape[2]] for x in c.held)
            NQ, hd = qb.shape
            rep = NQ // k.shape[1]
            for h in range(NQ):
                kh, vh = k[:, h // rep], v[:, h // rep]
                z = kh @ qb[h] * scale
                d = (kh.abs() @ qb[h].abs()).amax() * scale * (hd + 8) * R.E + 2.0 ** -21
                p = torch.exp(z - z.amax())
                tot = p.sum()
                A = p @ vh.abs() / tot
                out[h] = p @ vh / tot
                bound[h] = R.U * out[h].abs() + (R.U + 2 * d + 3 * n * R.E) * A + R.TINY + n * 2.0 ** -37 * vh.abs().amax() / tot
        outs.append(out)
        bounds.append(bound)
    return torch.stack(outs), torch.stack(bounds)


def run(c, table, lens, cu, shared, q, **kw):
    return ops.kv4_shared_attention(q, *c, table, lens, cu, shared, **kw)


def queries(dev, B, NQ, hd, seed):
    return torch.randn(B, NQ, hd, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).half()


GROUPS = [
    [(64, [1])],
    [(0, [5, 70])],
    [(128, [1, 64, 65]), (0, [3]), (192, [17, 300])],
    [(512, [30] * 9)],
    [(1024, [0, 1, 2, 3, 200])],
    [(64, [10] * 40), (2048, [100] * 3), (256, [0, 0])],
]


@pytest.mark.parametrize("hd,gs,page", [(64, 32, 16), (64, 64, 64), (128, 32, 32), (128, 64, 64), (128, 128, 16), (256, 32, 64),
                                        (256, 64, 16), (256, 128, 64)])
@pytest.mark.parametrize("NQ,NKV", [(4, 2), (14, 2), (8, 8)])
@pytest.mark.parametrize("groups", range(len(GROUPS)))
def test_groups(cuda, groups, NQ, NKV, hd, gs, page):
    c, table, lens, cu, shared = scene(cuda, GROUPS[groups], NKV, hd, gs, page, groups + hd)
    q = queries(cuda, len(lens), NQ, hd, groups)
    got = run(c, table, lens, cu, shared, q)
    ref, bound = reference(c, table, lens, q, 1 / math.sqrt(hd))
    R.assert_within(got, ref, bound, "shared")
    tight = run(c, table, lens, cu, shared, q, max_len=max(1, int(lens.max())), max_shared=int(shared.max()))
    R.assert_within(tight, ref, bound, "with bounds")


@pytest.mark.parametrize("NQ,NKV", [(64, 1), (40, 1), (33, 1), (12, 1), (1, 1), (64, 8), (65, 13)])
@pytest.mark.parametrize("B", [1, 7, 50])
def test_head_layouts(cuda, NQ, NKV, B):
    """Columns that end inside a tile, more heads of a KV head than a tile holds, every number of waves side by side."""
    rng = np.random.RandomState(NQ + B)
    c, table, lens, cu, shared = scene(cuda, [(384, list(rng.randint(0, 150, B)))], NKV, 64, 64, 32, NQ)
    q = queries(cuda, B, NQ, 64, B)
    ref, bound = reference(c, table, lens, q, 0.2)
    R.assert_within(run(c, table, lens, cu, shared, q, scale=0.2), ref, bound, "heads")


@pytest.mark.parametrize("page", [16, 256])
def test_long_contexts_are_split(cuda, page):
    c, table, lens, cu, shared = scene(cuda, [(20480, [100, 3000, 7]), (256, [5000])], 2, 128, 64, page, 3)
    q = queries(cuda, 4, 8, 128, 1)
    ref, bound = reference(c, table, lens, q, 1 / math.sqrt(128))
    R.assert_within(run(c, table, lens, cu, shared, q), ref, bound, "long")


def test_lengths_that_disagree(cuda):
    """Shared lengths that are no multiple of 64, past a sequence's length, negative, different in a group, of empty and absent
    sequences: the answer is that of the tables."""
    c, table, lens, cu, shared = scene(cuda, [(1024, [50, 60, 70, 80, 90, 100]), (512, [9, 300])], 2, 64, 32, 64, 5)
    q = queries(cuda, 8, 4, 64, 2)
    for case in ([1000, 999, 64, 63, 0, 1024, 512, 512], [1024] * 6 + [512] * 2, [1 << 30] * 8, [-5] * 8, [128, 0, 0, 0, 0, 700, 1, 512]):
        for change in ({}, {1: 0}, {0: 30, 6: 0}, {2: -7, 3: 64, 7: 512}):
            ln = lens.clone()
            for b, n in change.items():
                ln[b] = n
            sh = torch.tensor(case, dtype=torch.int32, device=cuda)
            if max(case) > 1024:  # only what the tables have in common may be named
                sh = torch.minimum(sh, torch.tensor([1024] * 6 + [512] * 2, dtype=torch.int32, device=cuda))
            ref, bound = reference(c, table, ln.clamp_min(0), q, 1 / 8)
            R.assert_within(run(c, table, ln, cu, sh, q), ref, bound, f"{case} {change}")


def test_offsets_that_leave_sequences_out(cuda):
    c, table, lens, cu, shared = scene(cuda, [(256, [5, 6, 7, 8, 9, 10])], 2, 64, 64, 64, 6)
    q = queries(cuda, 6, 4, 64, 3)
    ref, bound = reference(c, table, lens, q, 1 / 8)
    for offsets in ([0], [0, 0], [2, 4], [0, 3, 6], [0, 6, 6, 6], [1, 1, 5], [0, 4, 2, 6], [0, 9], [-1, 6], [6, 0], [5, 6, 7]):
        cu = torch.tensor(offsets, dtype=torch.int32, device=cuda)
        R.assert_within(run(c, table, lens, cu, shared, q), ref, bound, f"offsets {offsets}")


def test_tokens_without_a_page(cuda):
    c, table, lens, cu, shared = scene(cuda, [(256, [100, 200, 90])], 2, 128, 64, 64, 7)
    q = queries(cuda, 3, 4, 128, 4)
    broken = table.clone()
    broken[:, 1] = -1                      # 64 of the shared tokens
    broken[1, 5] = 1 << 20                 # and 64 of one sequence's own
    got = run(c, broken, lens, cu, shared, q)
    for b in range(3):
        keep = [i for i in range(table.shape[1]) if 0 <= broken[b, i] < c[0].shape[0]]
        n = int(lens[b]) - 64 * (1 + (b == 1))
        t = table[b:b + 1, keep].contiguous()
        ref, bound = reference(c, t, torch.tensor([n], dtype=torch.int32, device=cuda), q[b:b + 1], 1 / math.sqrt(128))
        R.assert_within(got[b:b + 1], ref, bound, f"sequence {b}")
    none = torch.full_like(table, -1)
    assert not run(c, none, lens, cu, shared, q).any()


def test_values_that_are_not_finite(cuda):
    """In a shared token's V: its group of dimensions of every sequence that shares it; in one sequence's own: of that one."""
    c, table, lens, cu, shared = scene(cuda, [(128, [40, 50]), (64, [30])], 2, 128, 32, 64, 8)
    q = queries(cuda, 3, 4, 128, 5)
    want = run(c, table, lens, cu, shared, q)
    for bad in (float("inf"), float("nan")):
        for b, pos, hit in ((0, 70, [0, 1]), (1, 140, [1]), (2, 3, [2])):
            vs = c[3].clone()
            vs[table[b, pos // 64], 1, 2, pos % 64] = bad
            vp = c[2].clone()
            got = run((c[0], c[1], vp, vs), table, lens, cu, shared, q)
            for o in range(3):
                if o in hit:
                    assert not torch.isfinite(got[o, 2:, 64:96]).any()
                    assert torch.equal(got[o, :2], want[o, :2]) and torch.equal(got[o, 2:, :64], want[o, 2:, :64])
                else:
                    assert torch.equal(got[o], want[o])


def test_large_scores_and_values(cuda):
    c, table, lens, cu, shared = scene(cuda, [(512, [100, 20])], 2, 64, 32, 64, 9, std=40.0)
    q = queries(cuda, 2, 4, 64, 6) * 4
    ref, bound = reference(c, table, lens, q, 1 / 8)
    R.assert_within(run(c, table, lens, cu, shared, q), ref, bound, "large")


def test_equal_to_sequences_that_stand_alone(cuda):
    """Sharing changes no result beyond rounding: against the same call with nothing shared, and kv4_decode_attention."""
    c, table, lens, cu, shared = scene(cuda, [(2048, [77] * 20), (640, [500] * 4)], 4, 128, 64, 64, 10)
    q = queries(cuda, 24, 16, 128, 7)
    got, alone = run(c, table, lens, cu, shared, q), run(c, table, lens, cu, torch.zeros_like(shared), q)
    ref, bound = reference(c, table, lens, q, 1 / math.sqrt(128))
    R.assert_within(got, ref, bound, "shared")
    R.assert_within(alone, ref, bound, "alone")
    apart = (got.double() - ops.kv4_decode_attention(q, *c, table, lens).double()).abs()
    assert (apart <= 2 * bound).all()  # (its bound is no wider: the same roundings)


def test_many_sequences(cuda):
    rng = np.random.RandomState(1)
    groups = [(64 * int(rng.randint(0, 4)), list(rng.randint(0, 90, rng.randint(1, 12)))) for _ in range(220)]
    c, table, lens, cu, shared = scene(cuda, groups, 1, 64, 64, 64, 11)
    q = queries(cuda, len(lens), 2, 64, 8)
    assert len(lens) > 1024
    got = run(c, table, lens, cu, shared, q)
    pick = torch.tensor(sorted(set(rng.randint(0, len(lens), 60)) | {0, 1023, 1024, len(lens) - 1}), device=cuda)
    ref, bound = reference(c, table[pick].contiguous(), lens[pick].contiguous(), q[pick], 1 / 8)
    R.assert_within(got[pick], ref, bound, "many")
    single = torch.arange(len(lens) + 1, dtype=torch.int32, device=cuda)  # as many groups as sequences
    R.assert_within(run(c, table, lens, single, shared, q)[pick], ref, bound, "groups of one")


def test_strided_queries_outputs_workspaces(cuda):
    c, table, lens, cu, shared = scene(cuda, [(256, [20, 30, 40])], 2, 64, 32, 64, 12)
    wide = torch.randn(3, 3 * 4 * 64 + 4, device=cuda).half()
    view = wide[:, 4:4 + 256].view(3, 4, 64)
    want = run(c, table, lens, cu, shared, view.contiguous())
    assert torch.equal(run(c, table, lens, cu, shared, view), want)
    n = _C.kv4_shared_attention_workspace_bytes(3, 1, 4, 2, 64, 296, 256)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=cuda)
    out = torch.full((3, 4, 64), float("nan"), device=cuda).half()
    run(c, table, lens, cu, shared, view, max_len=296, max_shared=256, out=out, workspace=ws)
    assert torch.equal(out, run(c, table, lens, cu, shared, view, max_len=296, max_shared=256))


def test_streams_and_graphs(cuda):
    c, table, lens, cu, shared = scene(cuda, [(512, [64] * 6), (256, [64] * 2)], 2, 128, 64, 64, 13)
    q = queries(cuda, 8, 8, 128, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(c, table, lens, cu, shared, q)
    side.synchronize()
    assert torch.equal(got, run(c, table, lens, cu, shared, q))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(c, table, lens, cu, shared, q)
    full = lens.clone()
    for i in range(4):  # other lengths, groups and queries at each replay
        lens.copy_(full - 13 * i)
        shared.fill_(256 if i % 2 else 192)
        q.copy_(queries(cuda, 8, 8, 128, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(c, table, lens, cu, shared, q))
        ref, bound = reference(c, table, lens, q, 1 / math.sqrt(128))
        R.assert_within(out, ref, bound, f"replay {i}")


def test_refusals(cuda):
    c, table, lens, cu, shared = scene(cuda, [(64, [5, 6])], 2, 64, 32, 64, 14)
    q = queries(cuda, 2, 4, 64, 1)
    ws = torch.empty(16, dtype=torch.uint8, device=cuda)
    bad = [
        lambda: run(c, table, lens, cu, shared, q.float()), lambda: run(c, table, lens, cu, shared, q[:1]),
        lambda: run(c, table, lens, cu, shared, q[:, :3].contiguous()), lambda: run(c, table, lens, cu, shared, q.transpose(1, 2)),
        lambda: run(c, table, lens, cu.long(), shared, q), lambda: run(c, table, lens, cu[:0], shared, q),
        lambda: run(c, table, lens, cu, shared[:1], q), lambda: run(c, table, lens, cu, shared.float(), q),
        lambda: run(c, table, lens, cu.cpu(), shared, q), lambda: run(c, table, lens, cu, shared, q, max_len=-1),
        lambda: run(c, table, lens, cu, shared, q, max_len=1 << 20), lambda: run(c, table, lens, cu, shared, q, max_len=64, max_shared=65),
        lambda: run(c, table, lens, cu, shared, q, scale=0.0), lambda: run(c, table, lens, cu, shared, q, scale=float("inf")),
        lambda: run(c, table, lens, cu, shared, q, out=q), lambda: run(c, table, lens, cu, shared, q, workspace=ws),
        lambda: run(c, table.expand(2, -1)[:, :1].t(), lens, cu, shared, q),
        lambda: run(c, table[:1].expand(3000, -1).contiguous(), lens[:1].expand(3000).contiguous(), cu,
                    shared[:1].expand(3000).contiguous(), q[:1].expand(3000, -1, -1).contiguous()),
        lambda: run(c, table, lens, torch.zeros(3000, dtype=torch.int32, device=cuda), shared, q),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was taken")
