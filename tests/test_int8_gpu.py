"""8-bit rows and their products against 64-bit references.

Tolerances, from the kernels' roundings (U = 2^-11 half a binary16 step, E = 2^-24 half a binary32 step, both relative,
TINY = 2^-25 half a step below binary16's normal range):
  * rows: scales are one binary32 rounding of a binary64 value, codes follow from binary64 quotients: both are compared for
    equality, but for codes whose quotient lies within 2^-40 of a border (binary64's own error, times the reductions);
  * linear: the integer sum is exact; its conversion, two products by scales and the residual's sum are binary32:
    4 E (|y| + |r|), then U |ref| + TINY;
  * gate_up: g and u carry 3 E each; |silu'| <= 1.1, exp, sum and quotient add 8 E: |u| (8 E |silu| + 3.3 E |g|) +
    4 E |silu u|, then U |ref| + TINY.
"""
import numpy as np
import pytest
import torch

from soinfer import ops
from soinfer.quant import formats

pytestmark = pytest.mark.gpu
U, E, TINY = 2.0 ** -11, 2.0 ** -24, 2.0 ** -25


def rows_ref(x, res, weight, eps):
    """x, res fp16 [T, H] -> (codes, quotients, fp32 scales, h) in binary64."""
    h = x if res is None else (x.float() + res.float()).half()
    n = h.double().cpu().numpy()
    if weight is not None:
        n = n / np.sqrt((n * n).mean(-1, keepdims=True) + eps) * weight.double().cpu().numpy()
    s = (np.abs(n).max(-1) / 127).astype(np.float32)
    quot = np.where(s[:, None] > 0, n / np.where(s > 0, s, 1).astype(np.float64)[:, None], 0)
    return np.clip(np.rint(quot), -127, 127), quot, s, h


def check_rows(got, ref):
    q, s = got
    codes, quot, scales, _ = ref
    assert np.array_equal(s.cpu().numpy(), scales)
    border = np.abs(np.abs(quot - np.floor(quot)) - 0.5) < 2.0 ** -40
    bad = (q.cpu().numpy() != codes) & ~(border & (np.rint(quot) != quot))
    assert not bad.any(), np.argwhere(bad)[:4]


@pytest.mark.parametrize("T,H", [(1, 16), (3, 496), (2, 512), (5, 528), (7, 1024), (4, 2032), (9, 2048), (2, 2064), (3, 4096),
                                 (2, 6144), (5, 8208), (1, 16384), (2, 20000), (1, 65536), (301, 896)])
def test_rows(cuda, T, H):
    g = torch.Generator(device=cuda).manual_seed(T * 7919 + H)
    x = (torch.randn(T, H, generator=g, device=cuda) * torch.exp(torch.randn(1, H, generator=g, device=cuda))).half()
    r = torch.randn(T, H, generator=g, device=cuda).half()
    w = (1 + 0.3 * torch.randn(H, generator=g, device=cuda)).half()
    check_rows(ops.quantize_int8(x), rows_ref(x, None, None, 0))
    check_rows(ops.quantize_int8(x, w, 1e-5), rows_ref(x, None, w, 1e-5))
    q, s, h = ops.add_rmsnorm_int8(x, r, w, 1e-6)
    ref = rows_ref(x, r, w, 1e-6)
    assert torch.equal(h, ref[3])
    check_rows((q, s), ref)
    q2, s2 = ops.quantize_int8(h, w, 1e-6)
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_rows_of_ties_zeros_and_strided_views(cuda):
    # s = 127 / 127 = 1: quotients are the values, many of them ties
    x = torch.zeros(4, 64, device=cuda)
    x[0] = torch.arange(64, device=cuda) - 31.5
    x[0, 0] = 127
    x[1] = (torch.arange(64, device=cuda) * 0.5 - 16) / 4
    x[1, 5] = 31.75
    x[3, 7] = 2.0 ** -24
    x = x.half()
    check_rows(ops.quantize_int8(x), rows_ref(x, None, None, 0))
    q, s = ops.quantize_int8(x)
    assert s[2] == 0 and not q[2].any()
    assert q[0, 1] == -30 and q[0, 2] == -30  # -30.5 and -29.5 to even
    wide = torch.randn(6, 3 * 160 + 1, device=cuda).half()
    for view in (wide[:, 1:161], wide[::2, 161:321], wide[5:, 321:]):
        w = torch.ones(160, device=cuda).half()
        for a, b in zip(ops.quantize_int8(view, w), ops.quantize_int8(view.contiguous(), w)):
            assert torch.equal(a, b)
        for a, b in zip(ops.add_rmsnorm_int8(view, view, w), ops.add_rmsnorm_int8(view.contiguous(), view.contiguous(), w)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("H", [64, 2048, 5120, 20000])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_rows_that_are_not_finite(cuda, H, bad):
    x = torch.randn(3, H, device=cuda).half()
    x[1, H // 2] = bad
    clean = x.clone()
    clean[1, H // 2] = 0
    w = torch.ones(H, device=cuda).half()
    for weight in (None, w):
        q, s = ops.quantize_int8(x, weight)
        q0, s0 = ops.quantize_int8(clean, weight)
        assert torch.equal(q[[0, 2]], q0[[0, 2]]) and torch.equal(s[[0, 2]], s0[[0, 2]])
        assert not q[1].any() and not torch.isfinite(s[1])
    W = torch.randint(-127, 128, (5, H), dtype=torch.int8, device=cuda)
    y = ops.int8_linear(q, s, W, torch.ones(5, device=cuda))
    assert torch.isnan(y[1]).all() and not torch.isnan(y[[0, 2]]).any()


def problem(cuda, T, K, N, seed, mats=1):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randint(-127, 128, (T, K), generator=g, device=cuda, dtype=torch.int8)
    xs = torch.rand(T, generator=g, device=cuda) * 0.02 + 1e-3
    ws = [torch.randint(-128, 128, (N, K), generator=g, device=cuda, dtype=torch.int8) for _ in range(mats)]
    ss = [torch.rand(N, 1, generator=g, device=cuda) * 2e-3 + 1e-5 for _ in range(mats)]
    return x, xs, ws, ss


def product(x, xs, w, s):
    return (x.double() @ w.double().t() * xs.double()[:, None] * s.double().view(-1)).cpu().numpy()


def check_linear(y, x, xs, w, s, res=None):
    p = product(x, xs, w, s)
    r = 0 if res is None else res.double().cpu().numpy()
    ref = p + r
    err = np.abs(y.double().cpu().numpy() - ref)
    over = err > 4 * E * (np.abs(p) + np.abs(r)) + U * np.abs(ref) * (1 + 2.0 ** -10) + TINY
    assert not over.any(), (np.argwhere(over)[:4], err.max())


def check_gate_up(h, x, xs, ws, ss):
    g, u = product(x, xs, ws[0], ss[0]), product(x, xs, ws[1], ss[1])
    silu = g / (1 + np.exp(-g))
    ref = silu * u
    err = np.abs(h.double().cpu().numpy() - ref)
    tol = np.abs(u) * (8 * E * np.abs(silu) + 3.3 * E * np.abs(g)) + 4 * E * np.abs(ref)
    over = err > tol + U * np.abs(ref) * (1 + 2.0 ** -10) + TINY
    assert not over.any(), (np.argwhere(over)[:4], err.max())


# both kernels, every tile and split rule; K that ends inside a 256-, 128- and 64-byte step; N that ends inside a tile
SHAPES = [(1, 16, 1), (1, 2048, 4096), (2, 48, 17), (5, 2048, 130), (16, 272, 64), (17, 6144, 333), (31, 80, 1000),
          (33, 1024, 2050), (48, 640, 20001), (49, 144, 36), (64, 2064, 4100), (64, 256, 70000), (65, 128, 128),
          (65, 16, 3), (100, 2048, 1000), (129, 400, 257), (256, 6144, 512), (300, 144, 6145), (777, 2048, 4096),
          (1025, 208, 4099), (2049, 1040, 8200), (4096, 112, 5000), (4000, 112, 4050), (4000, 208, 2040), (3850, 80, 4090),
          (200, 48, 2072), (40, 6144, 2040)]


@pytest.mark.parametrize("T,K,N", SHAPES)
def test_linear(cuda, T, K, N):
    x, xs, (w,), (s,) = problem(cuda, T, K, N, T + K + N)
    y = ops.int8_linear(x, xs, w, s)
    check_linear(y, x, xs, w, s)
    res = torch.randn(T, N, device=cuda).half() * 8
    z = ops.int8_linear(x, xs, w, s.view(-1), residual=res)
    check_linear(z, x, xs, w, s, res)
    out = res.clone()
    ops.int8_linear(x, xs, w, s, residual=out, out=out)
    assert torch.equal(out, z)


@pytest.mark.parametrize("T,K,N", [s for s in SHAPES if s[2] < 20000])
def test_gate_up(cuda, T, K, N):
    x, xs, ws, ss = problem(cuda, T, K, N, T * K + N, mats=2)
    check_gate_up(ops.int8_gate_up(x, xs, ws[0], ss[0], ws[1], ss[1]), x, xs, ws, ss)


def test_largest_sums_are_exact(cuda):
    """All codes at their largest: sums next to 2^31."""
    K = 131056
    for T in (3, 70):
        x = torch.full((T, K), -128, dtype=torch.int8, device=cuda)
        w = torch.full((5, K), -128, dtype=torch.int8, device=cuda)
        w[1] = 127
        one = torch.ones(T, device=cuda)
        y = ops.int8_linear(x, one, w, torch.full((5,), 2.0 ** -16, device=cuda))
        want = torch.tensor([K * 16384, -K * 16256, K * 16384, K * 16384, K * 16384], dtype=torch.float64) * 2.0 ** -16
        assert torch.equal(y.cpu(), want.half().expand(T, 5))


def test_a_row_does_not_depend_on_the_batch(cuda):
    """Exact sums: the same row gives the same bits through every tile and split."""
    x, xs, (w,), (s,) = problem(cuda, 700, 1040, 515, 3)
    y = ops.int8_linear(x, xs, w, s)
    for n in (1, 17, 40, 64, 65, 200):
        assert torch.equal(ops.int8_linear(x[:n], xs[:n], w, s), y[:n])


def test_rows_far_apart(cuda):
    """Weights and outputs past 2^31 elements."""
    N, K, T = 270001, 8192, 3
    w = torch.randint(-127, 128, (N, K), dtype=torch.int8, device=cuda)
    s = torch.full((N,), 1e-3, device=cuda)
    x, xs, _, _ = problem(cuda, T, K, 1, 5)
    y = ops.int8_linear(x, xs, w, s)
    check_linear(y[:, -300:], x, xs, w[-300:], s[-300:])
    T = 8500
    x, xs, _, _ = problem(cuda, T, 16, 1, 6)
    w = w.view(-1)[:N * 16].view(N, 16)
    y = ops.int8_linear(x, xs, w, s)
    check_linear(y[-200:, -300:].contiguous(), x[-200:], xs[-200:], w[-300:], s[-300:])


def test_quantizer_s_rows_and_unaligned_outputs(cuda):
    W = torch.randn(130, 512, device=cuda) * 0.02
    qt = formats.quantize(W, formats.QuantConfig(8, "per_channel"))
    x = torch.randn(70, 512, device=cuda).half()
    q, s = ops.quantize_int8(x)
    for T in (9, 70):
        buf = torch.full((T * 128 + 8,), float("nan"), dtype=torch.float16, device=cuda)
        out = buf[1:1 + T * 128].view(T, 128)  # 2-byte aligned
        ops.int8_linear(q[:T], s[:T], qt.qweight[:128], qt.scale[:128].contiguous(), out=out)
        check_linear(out, q[:T], s[:T], qt.qweight[:128], qt.scale[:128])
        assert torch.isnan(buf[0]) and torch.isnan(buf[1 + T * 128:]).all()  # nothing behind it
        assert torch.equal(out, ops.int8_linear(q[:T], s[:T], qt.qweight[:128], qt.scale[:128].contiguous()))


def test_no_rows(cuda):
    w, s = torch.zeros(8, 32, dtype=torch.int8, device=cuda), torch.ones(8, device=cuda)
    x = torch.zeros(0, 32, device=cuda).half()
    q, sc = ops.quantize_int8(x, torch.ones(32, device=cuda).half())
    assert q.shape == (0, 32) and sc.shape == (0,)
    assert ops.int8_linear(q, sc, w, s).shape == (0, 8)
    assert ops.int8_gate_up(q, sc, w, s, w, s).shape == (0, 8)
    assert ops.add_rmsnorm_int8(x, x, torch.ones(32, device=cuda).half())[2].shape == (0, 32)


def test_refusals(cuda):
    x, xs, (w, up), (s, us) = problem(cuda, 4, 64, 8, 1, mats=2)
    h = torch.randn(4, 64, device=cuda).half()
    wt = torch.ones(64, device=cuda).half()
    bad = [
        lambda: ops.quantize_int8(h[:, :40]),                       # not a multiple of 16
        lambda: ops.quantize_int8(h.float()),
        lambda: ops.quantize_int8(h.t()),
        lambda: ops.quantize_int8(h.view(-1)),
        lambda: ops.quantize_int8(h[:1].expand(4, 64)),             # rows on one another
        lambda: ops.quantize_int8(h, wt[:32]),
        lambda: ops.quantize_int8(h, wt, -1.0),
        lambda: ops.quantize_int8(h.cpu()),
        lambda: ops.add_rmsnorm_int8(h, h[:3], wt),
        lambda: ops.add_rmsnorm_int8(h, h.cpu(), wt),
        lambda: ops.int8_linear(x[:, :40].contiguous(), xs, w[:, :40].contiguous(), s),
        lambda: ops.int8_linear(x[:, :32], xs, w[:, :32].contiguous(), s),  # not contiguous
        lambda: ops.int8_linear(x, xs, w[:, :32].contiguous(), s),
        lambda: ops.int8_linear(x, xs[:3], w, s),
        lambda: ops.int8_linear(x, xs, w, s[:7]),
        lambda: ops.int8_linear(x, xs, w, s.view(1, 8)),
        lambda: ops.int8_linear(x.float(), xs, w, s),
        lambda: ops.int8_linear(x, xs.half(), w, s),
        lambda: ops.int8_linear(x, xs, w, s, residual=torch.zeros(4, 7, device=cuda).half()),
        lambda: ops.int8_linear(x, xs, w, s, out=torch.zeros(4, 8, device=cuda)),
        lambda: ops.int8_linear(x, xs, w, s, out=torch.zeros(8, 4, device=cuda).half().t()),
        lambda: ops.int8_linear(x.view(-1)[8:136].view(2, 64), xs[:2], w, s),  # 8-byte aligned
        lambda: ops.int8_gate_up(x, xs, w, s, up[:4].contiguous(), us[:4].contiguous()),
        lambda: ops.int8_gate_up(x, xs, w, s, up, us[:4].contiguous()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was taken")
    res = torch.zeros(9, 4, device=cuda).half()
    with pytest.raises(RuntimeError, match="overlap"):
        ops.int8_linear(x, xs, w, s, residual=res.view(-1)[:32].view(4, 8), out=res.view(-1)[4:36].view(4, 8))


def test_streams_and_graphs(cuda):
    x, xs, ws, ss = problem(cuda, 40, 512, 384, 9, mats=2)
    h, w = torch.randn(40, 512, device=cuda).half(), torch.ones(512, device=cuda).half()

    def calls():
        q, s, t = ops.add_rmsnorm_int8(h, h, w)
        return q, s, t, ops.int8_linear(q, s, ws[0], ss[0]), ops.int8_gate_up(q, s, ws[0], ss[0], ws[1], ss[1])

    want = [t.clone() for t in calls()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = calls()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for _ in range(3):
        h.copy_(torch.randn(40, 512, device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, calls()))


# the tiles of three stages: rows of one tile, tiles that fit the CUs once, eight waves; each way of storing
@pytest.mark.parametrize("T,K,N", [(64, 1040, 9000), (33, 272, 16385), (1, 64, 20004), (130, 400, 6000), (520, 208, 5004),
                                   (520, 208, 2500), (500, 144, 2051), (250, 2064, 4104), (700, 16, 3000), (511, 6144, 4099)])
def test_tiles_of_three_stages(cuda, T, K, N):
    x, xs, ws, ss = problem(cuda, T, K, N, T * K + 3 * N, mats=2)
    res = torch.randn(T, N, device=cuda).half() * 8
    check_linear(ops.int8_linear(x, xs, ws[0], ss[0], residual=res), x, xs, ws[0], ss[0], res)
    check_gate_up(ops.int8_gate_up(x, xs, ws[0], ss[0], ws[1], ss[1]), x, xs, ws, ss)
    # a row alone, through another tile, has the same bits
    t = T // 2
    row = ops.int8_gate_up(x[t:t + 1], xs[t:t + 1], ws[0], ss[0], ws[1], ss[1])
    assert torch.equal(row, ops.int8_gate_up(x, xs, ws[0], ss[0], ws[1], ss[1])[t:t + 1])
