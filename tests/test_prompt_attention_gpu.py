"""Causal attention of packed prompts (ops.prompt_attention) against the formula in 64 bits."""
import math

import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu


def problem(dev, nq, nk, NQ, NKV, hd, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda n, h: (torch.randn((n, h, hd), generator=g, device=dev) * scale).half()  # noqa: E731
    cu = [torch.from_numpy(R.offsets(x)).to(dev) for x in (nq, nk)]
    return mk(sum(nq), NQ), mk(sum(nk), NKV), mk(sum(nk), NKV), *cu


def check(got, q, k, v, nq, nk, label, scale=None):
    q0 = k0 = 0
    scale = scale or 1 / math.sqrt(q.shape[2])
    for i, (a, b) in enumerate(zip(nq, nk)):
        last = torch.arange(a, device=q.device) + b - a
        ref, bound = R.attention(q[q0:q0 + a].double(), k[k0:k0 + b].double(), v[k0:k0 + b].double(), last, scale)
        R.assert_within(got[q0:q0 + a], ref, bound, f"{label} sequence {i}")
        q0, k0 = q0 + a, k0 + b


@pytest.mark.parametrize("hd", [8, 40, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("NQ,NKV", [(4, 4), (6, 2), (8, 1)])
def test_head_layouts(cuda, hd, NQ, NKV):
    import soinfer.ops as ops

    n = [1, 31, 32, 33, 63, 64, 65, 129, 200]
    q, k, v, cu, _ = problem(cuda, n, n, NQ, NKV, hd, hd + NQ)
    check(ops.prompt_attention(q, k, v, cu, cu, max(n)), q, k, v, n, n, f"hd {hd}")


@pytest.mark.parametrize("nq,nk", [([1], [1]), ([1], [700]), ([5, 0, 3], [5, 4, 900]), ([127, 128, 257], [300, 128, 1000]),
                                   ([600], [601]), ([0, 2], [0, 2]), ([2000], [2000])])
def test_lengths(cuda, nq, nk):
    import soinfer.ops as ops

    q, k, v, cu_q, cu_k = problem(cuda, nq, nk, 4, 2, 128, 5, 1.5)
    check(ops.prompt_attention(q, k, v, cu_q, cu_k, max(nq)), q, k, v, nq, nk, f"{nq} {nk}")


@pytest.mark.parametrize("hd", [40, 64, 128, 200])
@pytest.mark.parametrize("nq,nk", [([1, 40, 0], [1500, 3000, 9]), ([130], [1100]), ([700, 5], [700, 5000]), ([3], [129])])
def test_split_keys(cuda, hd, nq, nk):
    """Few queries: their keys are split over workgroups, some rows' more than others'."""
    import soinfer._C as _C
    import soinfer.ops as ops

    q, k, v, cu_q, cu_k = problem(cuda, nq, nk, 4, 2, hd, 12)
    n = _C.prompt_attention_workspace_bytes(sum(nq), sum(nk), 4, hd)
    # 129 keys are fewer than two splits of four tiles where a tile has 64 keys (head_dim up to 64, or over 128)
    assert n > 0 or (nk == [129] and not 64 < hd <= 128)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device=cuda)  # NaN floats: what it held before does not matter
    out = torch.full_like(q, 2.0)
    ops.prompt_attention(q, k, v, cu_q, cu_k, max(nq), out=out, workspace=ws)
    check(out, q, k, v, nq, nk, f"split {hd}")
    assert torch.equal(out, ops.prompt_attention(q, k, v, cu_q, cu_k, max(nq) + 500))
    if n:
        with pytest.raises(RuntimeError, match="workspace"):
            ops.prompt_attention(q, k, v, cu_q, cu_k, max(nq), workspace=ws[:n - 16])


def test_queries_without_keys_give_zeros(cuda):
    import soinfer.ops as ops

    nq, nk = [40, 70, 3], [10, 0, 3]
    q, k, v, cu_q, cu_k = problem(cuda, nq, nk, 4, 2, 64, 6)
    got = ops.prompt_attention(q, k, v, cu_q, cu_k, 70)
    check(got, q, k, v, nq, nk, "short keys")
    assert (got[:30] == 0).all() and (got[40:110] == 0).all()


@pytest.mark.parametrize("NQ,NKV", [(2, 2), (2, 1), (4, 1), (14, 2)])
def test_no_keys_at_all(cuda, NQ, NKV):
    import soinfer.ops as ops

    q, _, _, cu_q, cu_k = problem(cuda, [40, 3], [0, 0], NQ, NKV, 64, 16)
    empty = torch.empty((0, NKV, 64), dtype=torch.float16, device=cuda)
    assert (ops.prompt_attention(q, empty, empty, cu_q, cu_k, 40) == 0).all()


@pytest.mark.parametrize("rep", [1, 2, 3, 4, 6, 7, 8, 12])
def test_heads_that_share_a_workgroup(cuda, rep):
    """Every part of a workgroup's queries, with and without a cached beginning, for each number of heads a KV head has."""
    import soinfer.ops as ops

    nq, nk = [1, 32, 33, 95, 128, 129, 200], [1, 40, 33, 300, 128, 777, 200]
    q, k, v, cu_q, cu_k = problem(cuda, nq, nk, 3 * rep, 3, 64, 17 + rep)
    check(ops.prompt_attention(q, k, v, cu_q, cu_k, 200), q, k, v, nq, nk, f"rep {rep}")


def test_strided_views_and_output(cuda):
    """q, k, v as views of one fused projection, the output into every other head of a wider tensor."""
    import soinfer.ops as ops

    NQ, NKV, hd, n = 6, 2, 64, [50, 77]
    g = torch.Generator(device=cuda).manual_seed(7)
    rows = torch.randn((sum(n), NQ + 2 * NKV, hd), generator=g, device=cuda).half()
    q, k, v = rows.split([NQ, NKV, NKV], 1)
    cu = torch.from_numpy(R.offsets(n)).to(cuda)
    out = torch.full((sum(n), 2 * NQ, hd), 7.0, dtype=torch.float16, device=cuda)
    got = ops.prompt_attention(q, k, v, cu, cu, 77, out=out[:, ::2])
    assert got.data_ptr() == out.data_ptr()
    check(out[:, ::2], q, k, v, n, n, "views")
    assert (out[:, 1::2] == 7).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_that_are_not_finite_reach_their_queries_only(cuda, hd):
    """An infinity or NaN in k or v is seen from its own position on; before it, and in the other sequence, every output
    is what it would be without it."""
    import soinfer.ops as ops

    n = [200, 90]
    q, k, v, cu, _ = problem(cuda, n, n, 4, 2, hd, 13)
    want = ops.prompt_attention(q, k, v, cu, cu, 200)
    for at, dim, bad in ((150, 5, math.inf), (150, hd - 1, -math.inf), (131, 33, math.nan), (199, 0, math.nan), (0, 1, math.inf)):
        v2 = v.clone()
        v2[at, 1, dim] = bad
        got = ops.prompt_attention(q, k, v2, cu, cu, 200)
        assert torch.equal(got[:at], want[:at]) and torch.equal(got[200:], want[200:]) and torch.equal(got[:, :2], want[:, :2])
        seen = got[at:200, 2:, dim].float()
        assert torch.isnan(seen).all() if math.isnan(bad) else ((seen == bad) | torch.isnan(seen)).all(), (at, bad)
        other = torch.arange(hd, device=cuda) != dim
        assert torch.equal(got[at:200, 2:, other], want[at:200, 2:, other])
        k2 = k.clone()
        k2[at, 1, dim] = bad
        got = ops.prompt_attention(q, k2, v, cu, cu, 200)
        assert torch.equal(got[:at], want[:at]) and torch.equal(got[200:], want[200:]) and torch.equal(got[:, :2], want[:, :2])
    v2 = v.clone()
    v2[140, 0, 7], v2[160, 0, 7] = math.inf, -math.inf
    got = ops.prompt_attention(q, k, v2, cu, cu, 200)
    assert torch.equal(got[:140], want[:140]) and torch.isnan(got[160:200, :2, 7]).all()


def test_rows_behind_the_last_sequence_stay(cuda):
    import soinfer.ops as ops

    n = [33, 20]
    q, k, v, cu, _ = problem(cuda, [33, 20, 90], [33, 20, 90], 4, 2, 128, 8)
    cu = cu[:3].contiguous()
    out = torch.full_like(q, 3.0)
    ops.prompt_attention(q, k, v, cu, cu, 33, out=out)
    check(out, q, k, v, n, n, "padded")
    assert (out[53:] == 3).all()


def test_large_scores_and_scale(cuda):
    import soinfer.ops as ops

    n = [150]
    q, k, v, cu, _ = problem(cuda, n, n, 2, 1, 128, 9, 12.0)
    check(ops.prompt_attention(q, k, v, cu, cu, 150), q, k, v, n, n, "large")
    check(ops.prompt_attention(q, k, v, cu, cu, 150, scale=0.01), q, k, v, n, n, "scale", 0.01)


def test_same_bits_again_and_in_a_graph(cuda):
    import soinfer.ops as ops

    n = [100, 300]
    q, k, v, cu, _ = problem(cuda, n, n, 8, 2, 128, 10)
    want = ops.prompt_attention(q, k, v, cu, cu, 300)
    assert torch.equal(want, ops.prompt_attention(q, k, v, cu, cu, 300))
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.prompt_attention(q, k, v, cu, cu, 300, out=out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(q, k, v, cu, cu, 300, out=out)
    for seed in range(3):
        q.copy_(problem(cuda, n, n, 8, 2, 128, 20 + seed)[0])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.prompt_attention(q, k, v, cu, cu, 300))


def test_rows_far_apart(cuda):
    """Offsets past 4 GiB: rows of q, k, v and out nearly 2^22 elements apart give the bits of contiguous ones."""
    import soinfer.ops as ops

    n, NQ, NKV, hd, stride = [300, 290], 4, 2, 64, (1 << 22) - 8
    q, k, v, cu, _ = problem(cuda, n, n, NQ, NKV, hd, 12)
    want = ops.prompt_attention(q, k, v, cu, cu, 300)
    base, outs = (torch.empty(sum(n) * stride, dtype=torch.float16, device=cuda) for _ in range(2))
    far = []
    for x, b, at in ((q, base, 0), (k, base, 4096), (v, base, 8192), (torch.zeros_like(q), outs, 0)):
        far.append(b.as_strided(x.shape, (stride, hd, 1), at))
        far[-1].copy_(x)
    ops.prompt_attention(*far[:3], cu, cu, 300, out=far[3])
    assert torch.equal(far[3], want)
    with pytest.raises(RuntimeError, match="apart"):
        ops.prompt_attention(q, base.as_strided((500, NKV, hd), (1 << 22, hd, 1)), v[:500], cu, cu, 300)


def test_rows_that_overlap(cuda):
    """One key row and one value row for all positions (stride 0): every query gets that value."""
    import soinfer.ops as ops

    n = [70]
    q, k, v, cu, _ = problem(cuda, n, n, 4, 2, 64, 13)
    k, v = k[:1].expand(70, -1, -1), v[:1].expand(70, -1, -1)
    check(ops.prompt_attention(q, k, v, cu, cu, 70), q, k, v, n, n, "one row")


def test_sequences_that_do_not_start_at_row_0(cuda):
    """cu starts behind rows of no sequence, which stay as they are, as do those behind the last."""
    import soinfer.ops as ops

    q, k, v, _, _ = problem(cuda, [100], [110], 4, 2, 128, 14)
    at = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    out = torch.full_like(q, 3.0)
    ops.prompt_attention(q, k, v, at(10, 40, 40, 90), at(20, 60, 60, 110), 50, out=out)
    check(out[10:90], q[10:90], k[20:110], v[20:110], [30, 0, 50], [40, 0, 50], "inner rows")
    assert (out[:10] == 3).all() and (out[90:] == 3).all()


def test_on_two_streams_at_once(cuda):
    """Calls with split keys that overlap on two streams, each with its own workspace, give what they give alone."""
    import soinfer.ops as ops

    q, k, v, cu_q, cu_k = problem(cuda, [60, 9], [2500, 700], 8, 2, 128, 15)
    q = [q, q.flip(0).contiguous()]
    want = [ops.prompt_attention(x, k, v, cu_q, cu_k, 60) for x in q]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.prompt_attention(q[i], k, v, cu_q, cu_k, 60))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_refusals(cuda):
    import soinfer.ops as ops

    n = [16]
    q, k, v, cu, _ = problem(cuda, n, n, 4, 2, 64, 11)
    bad = [
        dict(q=q.float()), dict(q=q.cpu()), dict(q=q[0]), dict(k=k[:, :1]), dict(k=k.transpose(1, 2)), dict(cu_q=cu.long()),
        dict(cu_k=cu[:1]), dict(max_q=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(out=q),
        dict(out=torch.empty_like(q)[:8]), dict(out=torch.empty_like(q).float()), dict(v=v[:8]),
    ]
    for change in bad:
        args = dict(q=q, k=k, v=v, cu_q=cu, cu_k=cu, max_q=16) | change
        with pytest.raises(RuntimeError):
            ops.prompt_attention(**args)
    flat = torch.zeros(16 * 2 * 64 + 4, dtype=torch.float16, device=cuda)
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.prompt_attention(q, flat[4:].view(16, 2, 64), v, cu, cu, 16)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ops.prompt_attention(q[..., :60], k[..., :60], v[..., :60], cu, cu, 16)
    with pytest.raises(RuntimeError, match="multiple of num_kv_heads"):
        ops.prompt_attention(q[:, :3], k, v, cu, cu, 16)
