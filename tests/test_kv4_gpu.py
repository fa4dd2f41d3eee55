"""The paged 4-bit KV cache on the GPU: append, read and single-token attention against the 64-bit definitions."""
import math

import numpy as np
import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu

SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


def table_of(lens, page, seed, extra=2):
    """Pages in any order, `extra` of them unused; entries behind a sequence's last page name no page."""
    counts = [-(-n // page) for n in lens]
    P = sum(counts) + extra
    order = np.random.RandomState(seed).permutation(P)
    table = np.full((len(lens), max(1, max(counts))), -1, np.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table, P


def filled(dev, lens, NKV, hd, gs, page, seed, fill=0xAB):
    """A cache with normal K and V, and the values it holds: (tensors, table, lens, [k, v] per sequence)."""
    rng = np.random.RandomState(seed)
    table, P = table_of(lens, page, seed)
    c = R.Cache(P, NKV, page, hd, gs, fill)
    c.ks[:], c.vs[:] = np.nan, np.nan  # slots that no token fills
    held = []
    for b, n in enumerate(lens):
        kv = rng.randn(2, n, NKV, hd).astype(np.float16)
        got = np.zeros(kv.shape)
        for t in range(n):
            for h in range(NKV):
                got[0, t, h], got[1, t, h] = c.put(table[b, t // page], h, t % page, kv[0, t, h], kv[1, t, h])
        held.append([torch.from_numpy(x).to(dev) for x in got])
    return c.tensors(dev), torch.from_numpy(table).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), held


# --------------------------------------------------------------------------- append

def append_problem(dev, olds, news, NQ, NKV, hd, gs, page, norm, seed, k_scale=1.0):
    rng = np.random.RandomState(seed)
    lens = [o + n for o, n in zip(olds, news)]
    table, P = table_of(lens, page, seed)
    T = sum(news)
    qkv = (rng.randn(T, (NQ + 2 * NKV) * hd) * k_scale).astype(np.float16)
    w = [(1 + 0.2 * rng.randn(hd)).astype(np.float16) for _ in range(2)] if norm else [None, None]
    cos, sin = R.rope_tables(max(lens), hd)
    return dict(qkv=qkv, w=w, cos=cos, sin=sin, table=table, P=P, lens=np.array(lens, np.int32), cu=R.offsets(news))


def append_ref(p, NQ, NKV, hd, gs, page, eps, limit=None):
    """(cache image, q exact, k exact), the image with 0x5C bytes and zero scales where nothing is appended."""
    c = R.Cache(p["P"], NKV, page, hd, gs, 0x5C)
    T = p["qkv"].shape[0]
    q, k = np.zeros((T, NQ, hd)), np.zeros((T, NKV, hd))
    rows = p["cos"].shape[0]
    for b in range(len(p["lens"])):
        lo, hi = int(p["cu"][b]), int(p["cu"][b + 1])
        for t in range(lo, hi):
            pos = int(p["lens"][b]) - (hi - t)
            x = p["qkv"][t].reshape(NQ + 2 * NKV, hd)
            r = min(max(pos, 0), rows - 1)
            q[t] = R.norm_rope(x[:NQ], p["w"][0], eps, p["cos"][r], p["sin"][r])
            k[t] = R.norm_rope(x[NQ:NQ + NKV], p["w"][1], eps, p["cos"][r], p["sin"][r])
            blk = pos // page
            if pos < 0 or pos >= rows or blk >= p["table"].shape[1] or not 0 <= p["table"][b, blk] < p["P"]:
                continue
            for h in range(NKV):
                c.put(p["table"][b, blk], h, pos % page, R.half(k[t, h]), x[NQ + NKV + h])
    return c, q, k


def run_append(dev, p, NQ, NKV, hd, gs, page, eps=1e-6, qkv=None):
    import soinfer.ops as ops

    c = R.Cache(p["P"], NKV, page, hd, gs, 0x5C).tensors(dev)
    up = lambda x: None if x is None else torch.from_numpy(x).to(dev)  # noqa: E731
    T = p["qkv"].shape[0]
    q_out = torch.full((T, NQ, hd), 9.0, dtype=torch.float16, device=dev)
    k_out = torch.full((T, NKV, hd), 9.0, dtype=torch.float16, device=dev)
    got = ops.kv4_append(up(p["qkv"]) if qkv is None else qkv, up(p["w"][0]), up(p["w"][1]), up(p["cos"]), up(p["sin"]), *c,
                         up(p["table"]), up(p["lens"]), up(p["cu"]), NQ, eps, k_out=k_out, q_out=q_out)
    assert got.data_ptr() == q_out.data_ptr()
    return c, q_out, k_out


def same_cache(c, ref):
    for got, want, name in zip(c, (ref.k, ref.ks, ref.v, ref.vs), ("k", "k_scale", "v", "v_scale")):
        R.same(got, want, name)


@pytest.mark.parametrize("hd,gs", SHAPES)
@pytest.mark.parametrize("norm", [False, True])
def test_append_bytes(cuda, hd, gs, norm):
    """Every byte of the cache, and q and k as the one rounding of the 64-bit rotation."""
    NQ, NKV, page = 6, 2, 16
    p = append_problem(cuda, [0, 5, 37, 3, 64], [9, 1, 0, 30, 17], NQ, NKV, hd, gs, page, norm, hd + gs + norm)
    ref, q, k = append_ref(p, NQ, NKV, hd, gs, page, 1e-6)
    c, qo, ko = run_append(cuda, p, NQ, NKV, hd, gs, page)
    same_cache(c, ref)
    R.same(qo, R.half(q), "q")
    R.same(ko, R.half(k), "k")


@pytest.mark.parametrize("B", [1, 3, 64, 65, 300])
def test_append_decode_steps(cuda, B):
    """One token per sequence, and the same with sequences that get none."""
    NQ, NKV, hd, gs, page = 4, 2, 128, 64, 32
    rng = np.random.RandomState(B)
    olds = rng.randint(0, 100, B).tolist()
    for news in ([1] * B, [int(x) for x in rng.randint(0, 3, B - 1)] + [2]):
        p = append_problem(cuda, olds, news, NQ, NKV, hd, gs, page, True, B)
        ref, q, _ = append_ref(p, NQ, NKV, hd, gs, page, 1e-6)
        c, qo, _ = run_append(cuda, p, NQ, NKV, hd, gs, page)
        same_cache(c, ref)
        R.same(qo, R.half(q), "q")


def test_append_values_at_borders(cuda):
    """Ties of the codes, scales below the normal range, zeros, the largest numbers, infinities and NaN."""
    NQ, NKV, hd, gs, page = 1, 1, 64, 32, 16
    rows = []
    ties = np.tile(np.array([7, 0.5, 1.5, 2.5, -0.5, -1.5, 3.5, 6.5], np.float16), 8)
    rows += [ties, ties * np.float16(2 ** -10), np.zeros(64, np.float16), np.full(64, 6e-8, np.float16)]
    rows += [np.full(64, 4e-7, np.float16), np.full(64, 65504, np.float16) * np.float16(-1)]
    for bad in (np.inf, -np.inf, np.nan):
        r = np.ones(64, np.float16)
        r[40] = bad
        rows.append(r)
    rng = np.random.RandomState(0)
    rows += [(rng.randint(-14, 15, 64) * 0.5 * 2.0 ** rng.randint(-20, 10)).astype(np.float16) for _ in range(23)]
    x = np.stack(rows)
    T = len(rows)
    p = append_problem(cuda, [0], [T], NQ, NKV, hd, gs, page, False, 1)
    p["qkv"] = np.concatenate([np.ones_like(x), x, x], 1)
    p["cos"], p["sin"] = np.ones((T, 32), np.float32), np.zeros((T, 32), np.float32)  # no turn
    c, _, _ = run_append(cuda, p, NQ, NKV, hd, gs, page)
    with np.errstate(invalid="ignore"):
        ref = append_ref(p, NQ, NKV, hd, gs, page, 1e-6)[0]
    for got, want, kind in ((c[0], ref.k, "k"), (c[2], ref.v, "v")):
        # a bad number spoils its own group of k's low half too (0 * inf in the rotation), so k is compared without them
        a, w = got.cpu().numpy(), want
        for t in range(T):
            if kind == "k" and not np.isfinite(x[t]).all():
                continue
            pg, slot = p["table"][0, t // page], t % page
            if kind == "k":
                R.same(a[pg, 0, slot], w[pg, 0, slot], f"k row {t}")
            else:
                ua = a[pg, 0].view(np.uint16).reshape(page // 4, 16, 1, 4)[slot // 4][..., slot % 4]
                uw = w[pg, 0].view(np.uint16).reshape(page // 4, 16, 1, 4)[slot // 4][..., slot % 4]
                R.same(ua, uw, f"v row {t}")
    import soinfer.ops as ops

    up = lambda a: torch.from_numpy(a).to(cuda)  # noqa: E731
    k, v = ops.kv4_read(*c, up(p["table"]), up(p["lens"]), up(p["cu"]), T)
    for i in range(6, 9):
        assert torch.isfinite(v[i, 0, :32]).all() and torch.isnan(v[i, 0, 32:]).all()


def test_append_outside_the_cache(cuda):
    """Missing pages, bad page numbers, positions past the block table, past the tables and below zero: nothing there is
    written, q is there all the same; rows behind the last sequence stay."""
    NQ, NKV, hd, gs, page = 4, 2, 128, 32, 16
    p = append_problem(cuda, [0, 20, 10, 0], [40, 30, 8, 4], NQ, NKV, hd, gs, page, True, 3)
    p["table"][0, 1] = -1
    p["table"][1, 1] = p["P"]
    p["table"][1, 2] = 1 << 30
    p["table"] = p["table"][:, :3]
    p["lens"][1] = 60  # positions 30 .. 59: past the 48 the table holds
    p["lens"][2] = 3   # positions -5 .. 2
    p["cos"], p["sin"] = p["cos"][:38], p["sin"][:38]
    p["cu"] = p["cu"][:4]  # the fourth sequence's rows are behind the last one
    p["lens"], p["table"] = p["lens"][:3], np.ascontiguousarray(p["table"][:3])
    ref, q, k = append_ref(p, NQ, NKV, hd, gs, page, 1e-6)
    c, qo, ko = run_append(cuda, p, NQ, NKV, hd, gs, page)
    same_cache(c, ref)
    n = int(p["cu"][3])
    R.same(qo[:n], R.half(q)[:n], "q")
    assert (qo[n:] == 9).all() and (ko[n:] == 9).all()


def test_append_strided_rows(cuda):
    """qkv as columns of a wider projection that start off a 16-byte boundary."""
    NQ, NKV, hd, gs, page = 4, 2, 64, 32, 16
    p = append_problem(cuda, [2, 7], [11, 4], NQ, NKV, hd, gs, page, True, 4)
    T, n = p["qkv"].shape
    wide = torch.zeros((T, n + 9), dtype=torch.float16, device=cuda)
    wide[:, 3:3 + n] = torch.from_numpy(p["qkv"]).to(cuda)
    ref, q, _ = append_ref(p, NQ, NKV, hd, gs, page, 1e-6)
    c, qo, _ = run_append(cuda, p, NQ, NKV, hd, gs, page, qkv=wide[:, 3:3 + n])
    same_cache(c, ref)
    R.same(qo, R.half(q), "q")


# --------------------------------------------------------------------------- read

@pytest.mark.parametrize("hd,gs", SHAPES)
def test_read(cuda, hd, gs):
    import soinfer.ops as ops

    lens = [1, 16, 47, 0, 33]
    c, table, lt, held = filled(cuda, lens, 3, hd, gs, 16, hd + gs)
    for ns in (lens, [1, 3, 40, 0, 17]):  # whole contexts, and the last positions of each
        cu = torch.from_numpy(R.offsets(ns)).to(cuda)
        T = sum(ns)
        k, v = ops.kv4_read(*c, table, lt, cu, T)
        want = [torch.cat([h[x][len(h[x]) - n:] for h, n in zip(held, ns)]) for x in (0, 1)]
        # code x scale is exact in binary32, so the binary16 value is one rounding of it
        assert torch.equal(k, want[0].float().half()) and torch.equal(v, want[1].float().half())


def test_read_outside_the_cache(cuda):
    import soinfer.ops as ops

    c, table, lt, held = filled(cuda, [40, 20], 2, 64, 32, 16, 5)
    table = table.clone()
    table[0, 1] = 10 ** 6
    cu = torch.tensor([0, 40, 65], dtype=torch.int32, device=cuda)  # 25 rows of a sequence of 20: positions -5 .. 19
    out = [torch.full((70, 2, 64), 4.0, dtype=torch.float16, device=cuda) for _ in range(2)]
    k, v = ops.kv4_read(*c, table, lt, cu, 70, *out)
    for got, x in ((k, 0), (v, 1)):
        want = held[0][x].float().half()
        want[16:32] = 0
        assert torch.equal(got[:40], want)
        assert (got[40:45] == 0).all() and torch.equal(got[45:65], held[1][x].float().half())
        assert (got[65:] == 4).all()


# --------------------------------------------------------------------------- attention

def check_attention(got, q, held, label, scale=None):
    scale = scale or 1 / math.sqrt(q.shape[2])
    for b, (k, v) in enumerate(held):
        last = torch.tensor([len(k) - 1], device=q.device)
        ref, bound = R.attention(q[b:b + 1].double(), k, v, last, scale)
        R.assert_within(got[b:b + 1], ref, bound, f"{label} sequence {b}")


def queries(dev, B, NQ, hd, seed, scale=1.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn((B, NQ, hd), generator=g, device=dev) * scale).half()


@pytest.mark.parametrize("hd,gs", SHAPES)
@pytest.mark.parametrize("NQ,NKV,page", [(2, 2, 16), (6, 2, 32), (20, 1, 64)])
def test_attention_layouts(cuda, hd, gs, NQ, NKV, page):
    import soinfer.ops as ops

    lens = [1, 15, 16, 17, 63, 64, 65, 0, 200]
    c, table, lt, held = filled(cuda, lens, NKV, hd, gs, page, hd + gs + NQ)
    q = queries(cuda, len(lens), NQ, hd, 1)
    got = ops.kv4_decode_attention(q, *c, table, lt, max_len=200)
    check_attention(got, q, held, f"hd {hd} gs {gs}")
    assert (got[7] == 0).all()


@pytest.mark.parametrize("L", [255, 256, 257, 1000, 2049])
def test_attention_split_lengths(cuda, L):
    """Contexts split over workgroups; the split follows max_len, the default being all the table holds."""
    import soinfer.ops as ops

    lens = [L, 3, L // 2]
    c, table, lt, held = filled(cuda, lens, 2, 64, 32, 64, L)
    q = queries(cuda, 3, 4, 64, L)
    for ml in (None, L, table.shape[1] * 64):
        check_attention(ops.kv4_decode_attention(q, *c, table, lt, max_len=ml), q, held, f"L {L} max_len {ml}")
    cut = ops.kv4_decode_attention(q, *c, table, lt, max_len=L // 2)  # no sequence is read past max_len
    check_attention(cut, q, [[x[:L // 2] for x in h] for h in held], "cut")


def test_attention_missing_pages(cuda):
    """Tokens without a page are left out, whatever the table says of them."""
    import soinfer.ops as ops

    c, table, lt, held = filled(cuda, [100, 40], 2, 128, 64, 16, 7)
    table = table.clone()
    table[0, 2], table[0, 5], table[1, 0] = -7, c[0].shape[0], -1
    keep = [torch.ones(100, dtype=torch.bool), torch.ones(40, dtype=torch.bool)]
    keep[0][32:48], keep[0][80:96], keep[1][:16] = False, False, False
    q = queries(cuda, 2, 4, 128, 7)
    got = ops.kv4_decode_attention(q, *c, table, lt)
    check_attention(got, q, [[x[m.to(cuda)] for x in h] for h, m in zip(held, keep)], "missing")
    lt2 = torch.tensor([10 ** 9, -3], dtype=torch.int32, device=cuda)  # lengths past the table, and below zero
    got2 = ops.kv4_decode_attention(q, *c, table, lt2, max_len=100)
    assert torch.equal(got2[0], got[0]) and (got2[1] == 0).all()


def test_attention_scale_stride_and_out(cuda):
    import soinfer.ops as ops

    c, table, lt, held = filled(cuda, [70, 300], 2, 128, 32, 32, 8)
    wide = queries(cuda, 2, 8, 128, 8)
    q = wide[:, 1:5]  # a token's heads are contiguous, its rows are not
    out = torch.empty((2, 4, 128), dtype=torch.float16, device=cuda)
    got = ops.kv4_decode_attention(q, *c, table, lt, scale=0.3, out=out)
    assert got.data_ptr() == out.data_ptr()
    check_attention(got, q, held, "scale", 0.3)


def test_attention_in_graphs_with_one_workspace(cuda):
    """Two captured steps share a workspace (replayed one after another); lengths and queries change between replays."""
    import soinfer._C as _C
    import soinfer.ops as ops

    c, table, lt, held = filled(cuda, [500, 129], 2, 64, 64, 64, 9)
    ws = torch.empty(_C.kv4_decode_attention_workspace_bytes(2, 4, 2, 64, 512), dtype=torch.uint8, device=cuda)
    ws.fill_(0xFF)  # NaN floats: what it held before does not matter
    q = [queries(cuda, 2, 4, 64, s) for s in (1, 2)]
    out = [torch.empty((2, 4, 64), dtype=torch.float16, device=cuda) for _ in q]
    run = lambda i: ops.kv4_decode_attention(q[i], *c, table, lt, max_len=512, out=out[i], workspace=ws)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(0)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(i)
        graphs.append(g)
    for lens in ([500, 129], [64, 1], [257, 0], [500, 129]):
        lt.copy_(torch.tensor(lens, dtype=torch.int32))
        for i, g in enumerate(graphs):
            q[i].copy_(queries(cuda, 2, 4, 64, 10 * i + lens[0]))
            out[i].fill_(5.0)
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            check_attention(out[i], q[i], [[x[:n] for x in h] for h, n in zip(held, lens)], f"replay {lens}")
            assert torch.equal(out[i], ops.kv4_decode_attention(q[i], *c, table, lt, max_len=512))


def test_pages_past_4_gib(cuda):
    """A cache whose K and V pages are 4.6 GB each: the same bytes and bits from its last pages as from a small one's."""
    import soinfer.ops as ops

    NQ, NKV, hd, gs, page, news = 8, 8, 128, 64, 64, [150, 1, 70]
    table, few = table_of(news, page, 3, extra=0)
    P = 140000
    up = lambda x: torch.from_numpy(x).to(cuda)  # noqa: E731
    p = append_problem(cuda, [0, 0, 0], news, NQ, NKV, hd, gs, page, True, 3)
    lens, cu = up(p["lens"]), up(p["cu"])

    def run(pages, at):
        c = [torch.empty((pages, NKV, page, hd // 2), dtype=torch.uint8, device=cuda),
             torch.empty((pages, NKV, hd // gs, page), dtype=torch.float16, device=cuda),
             torch.empty((pages, NKV, page, hd // 2), dtype=torch.uint8, device=cuda),
             torch.empty((pages, NKV, hd // gs, page), dtype=torch.float16, device=cuda)]
        for x in c:
            x[at:at + few].fill_(7)
        t = up(np.where(table < 0, -1, table + at).astype(np.int32))
        q = ops.kv4_append(up(p["qkv"]), up(p["w"][0]), up(p["w"][1]), up(p["cos"]), up(p["sin"]), *c, t, lens, cu, NQ)
        return [q, *ops.kv4_read(*c, t, lens, cu, sum(news)),
                ops.kv4_decode_attention(q[cu[1:].long() - 1], *c, t, lens, max_len=150), *(x[at:at + few].clone() for x in c)]

    for got, want in zip(run(P, P - few), run(few, 0)):
        R.same(got, want.cpu().numpy(), "far pages")


def test_on_two_streams_at_once(cuda):
    """Calls that overlap on two streams, each with its own workspace, give what they give alone."""
    import soinfer.ops as ops

    c, table, lt, held = filled(cuda, [900, 40, 300], 2, 128, 64, 64, 10)
    q = [queries(cuda, 3, 8, 128, s) for s in (1, 2)]
    want = [ops.kv4_decode_attention(x, *c, table, lt, max_len=900) for x in q]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.kv4_decode_attention(q[i], *c, table, lt, max_len=900))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_two_sequences_of_the_same_pages(cuda):
    """A shared beginning: two sequences name the same pages, and a third ends inside them."""
    import soinfer.ops as ops

    c, table, lt, held = filled(cuda, [130], 2, 64, 32, 16, 11)
    table, lt = table.expand(3, -1).contiguous(), torch.tensor([130, 130, 50], dtype=torch.int32, device=cuda)
    q = queries(cuda, 1, 4, 64, 3).expand(3, -1, -1).contiguous()
    got = ops.kv4_decode_attention(q, *c, table, lt, max_len=130)
    check_attention(got, q, [held[0], held[0], [x[:50] for x in held[0]]], "shared pages")
    assert torch.equal(got[0], got[1])


def test_refusals(cuda):
    import soinfer.ops as ops

    c, table, lt, _ = filled(cuda, [20, 9], 2, 64, 32, 16, 11)
    q = queries(cuda, 2, 4, 64, 11)
    ok = dict(q=q, k_pages=c[0], k_scale=c[1], v_pages=c[2], v_scale=c[3], block_table=table, seq_lens=lt)
    ops.kv4_decode_attention(**ok)
    for change in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:1]), dict(q=q[..., :32]), dict(q=q.transpose(1, 2)),
                   dict(q=q[:, :3]), dict(k_pages=c[0].int()), dict(k_pages=c[0][:, :1]), dict(k_scale=c[1][..., :8]),
                   dict(k_scale=c[1].float()), dict(v_scale=c[3][:, :, :1]), dict(block_table=table.long()),
                   dict(block_table=table[:1]), dict(seq_lens=lt.cpu()), dict(max_len=-1), dict(max_len=1 << 20),
                   dict(out=q), dict(out=q[:1].clone()), dict(scale=float("nan"))):
        with pytest.raises(RuntimeError):
            ops.kv4_decode_attention(**(ok | change))
    big = filled(cuda, [600], 2, 64, 32, 16, 12)
    with pytest.raises(RuntimeError, match="workspace"):
        ops.kv4_decode_attention(q[:1], *big[0], big[1], big[2], workspace=torch.empty(8, dtype=torch.uint8, device=cuda))
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    qkv = torch.zeros((2, 8 * 64), dtype=torch.float16, device=cuda)
    cos = torch.ones((32, 32), device=cuda)
    w = torch.ones(64, dtype=torch.float16, device=cuda)
    ok = dict(qkv=qkv, q_norm=w, k_norm=w, cos_table=cos, sin_table=cos, k_pages=c[0], k_scale=c[1], v_pages=c[2],
              v_scale=c[3], block_table=table, seq_lens=lt, cu_seqlens=cu, num_q_heads=4)
    ops.kv4_append(**ok)
    for change in (dict(qkv=qkv.float()), dict(qkv=qkv[:, :-64]), dict(qkv=qkv.t()), dict(q_norm=None), dict(q_norm=w[:32]),
                   dict(cos_table=cos[:, :16]), dict(sin_table=cos.half()), dict(cu_seqlens=cu[:2]),
                   dict(cu_seqlens=cu.long()), dict(num_q_heads=5), dict(num_q_heads=0),
                   dict(q_out=qkv.view(2, 8, 64)[:, :4]), dict(k_out=torch.zeros((2, 4, 64), device=cuda).half())):
        with pytest.raises(RuntimeError):
            ops.kv4_append(**(ok | change))
    for change in (dict(num_tokens=-1), dict(cu_seqlens=cu[1:]), dict(k_out=w), dict(k_pages=c[0].cpu())):
        args = dict(k_pages=c[0], k_scale=c[1], v_pages=c[2], v_scale=c[3], block_table=table, seq_lens=lt, cu_seqlens=cu,
                    num_tokens=2) | change
        with pytest.raises(RuntimeError):
            ops.kv4_read(**args)
