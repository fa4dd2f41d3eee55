"""sample_tokens against a 64-bit row-by-row reference in Python integers and numpy.

Tokens have to be equal. The reference's weights are exact to 2^-52, the kernel's to 2^-44 of the largest, so a border (top-p,
min-p or the drawn token's) can fall differently only where it lies within V 2^-43 of a token's: `close` finds those rows
from the reference alone (none in these inputs but the ones made for it), and they may take either neighbour.
"""
import numpy as np
import pytest
import torch

from soinfer import _C, ops

pytestmark = pytest.mark.gpu


def reference(l, u, T, k, p, m):
    """(token, the tokens that a border within V 2^-43 also allows)."""
    l = l.astype(np.float64)
    u, T, p, m = (float(np.float32(x)) for x in (u, T, p, m))
    if np.isnan(l).any():
        t = int(np.flatnonzero(np.isnan(l))[0])
        return t, {t}
    if not T > 0 or not np.isfinite(l.max()):
        t = int(np.argmax(l))
        return t, {t}
    order = np.argsort(-l, kind="stable")
    order = order[np.isfinite(l[order])]
    w = np.exp((l[order] - l[order[0]]) / T)
    near = len(l) * 2.0 ** -43
    if k > 0:
        order, w = order[:k], w[:k]
    answers = set()
    token = None
    for dp in (0, -1, 1):
        for dm in (0, -1, 1):
            o, v = order, w
            if p < 1:
                front = np.concatenate([[0], np.cumsum(v)[:-1]])
                n = max(1, int((front < p * v.sum() + dp * near).sum()))
                o, v = o[:n], v[:n]
            if m > 0:
                ok = v >= min(m, 1.0) * (1 + dm * 1e-14)
                ok[0] = True
                o, v = o[ok], v[ok]
            cum = np.cumsum(v)
            for du in (0, -1, 1):
                n = int((cum <= min(max(u, 0), 1) * cum[-1] + du * near).sum())
                t = int(o[min(n, int((v > 2.0 ** -45).sum()) - 1)])
                answers.add(t)
                if dp == dm == du == 0:
                    token = t
    return token, answers


def check(logits, u, T, k, p, m, close_allowed=0.02, **kw):
    got = ops.sample_tokens(logits, u, T, k, p, m, **kw).cpu().numpy()
    B = logits.shape[0]

    def row(x, b):
        return x[b].item() if isinstance(x, torch.Tensor) else x

    close = 0
    lc = logits.float().cpu().numpy()
    for b in range(B):
        want, also = reference(lc[b], u[b].item(), row(T, b), row(k, b), row(p, b), row(m, b))
        close += len(also) > 1
        assert got[b] in also, (b, got[b], want, also, row(T, b), row(k, b), row(p, b), row(m, b))
    assert close <= max(1, close_allowed * B), "the reference leaves too many rows open"
    return got


def rows(cuda, B, V, seed, spread=2.5, half=True):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn(B, V, generator=g, device=cuda) * spread
    x.scatter_add_(1, torch.randint(0, V, (B, 5), generator=g, device=cuda), torch.full((B, 5), 2 * spread, device=cuda))
    return (x.half() if half else x), torch.rand(B, generator=g, device=cuda)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.02),
            (1.0, 5000, 0.8, 0.0), (1.0, 3000, 1.0, 0.001), (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.05, 0.0),
            (1.0, 0, 0.99, 0.3), (2.0, 0, 0.999, 1e-4), (1.0, 10 ** 9, 0.5, 0.0), (1.0, 7, 0.5, 1.0)]


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 1023, 8191, 8192, 8193, 32000, 50257, 151936])
def test_settings(cuda, V, half):
    for i, s in enumerate(SETTINGS):
        x, u = rows(cuda, 3, V, V + i, half=half)
        check(x, u, *s)


@pytest.mark.parametrize("spread", [0.05, 0.5, 1.5, 4.0, 12.0])
def test_distributions_and_row_settings(cuda, spread):
    """Each row its own settings; flat to peaked; several chunks a row, one and many rows."""
    r = np.random.default_rng(int(spread * 100))
    for B, V in ((1, 40000), (70, 20011), (300, 1500)):
        x, u = rows(cuda, B, V, B, spread)
        T = torch.tensor(r.choice([0.0, 0.3, 1.0, 1.7], B), dtype=torch.float32, device=cuda)
        k = torch.tensor(r.choice([-1, 0, 1, 20, 2048, 2049, 9000], B), dtype=torch.int32, device=cuda)
        p = torch.tensor(r.choice([1.0, 0.3, 0.9, 0.999, 1.5], B), dtype=torch.float32, device=cuda)
        m = torch.tensor(r.choice([0.0, 0.01, 0.2, -1.0], B), dtype=torch.float32, device=cuda)
        check(x, u, T, k, p, m)


def test_equal_logits(cuda):
    """More equal logits than the list of collected tokens holds: every rule cuts in the middle of them, lower index first."""
    V = 60000
    x = torch.zeros(4, V, device=cuda).half()
    x[1] = -5.0
    x[1, 100] = x[1, 59999] = 1.0
    x[2, ::2] = -0.0  # the same number as 0
    x[3, 1::3] = -1.0
    u = torch.tensor([0.25, 0.9, 0.5, 0.999], device=cuda)
    for s in SETTINGS:
        check(x, u, *s, close_allowed=1)
    got = ops.sample_tokens(x, u, 1.0, 30000, 0.5)
    assert got[0] == 3750 and got[2] == 7500  # floor(u 15000)
    assert ops.sample_tokens(x[:1], u[2:3])[0] == 30000


def test_random_numbers_at_their_ends(cuda):
    x, _ = rows(cuda, 6, 3001, 1)
    last = torch.tensor([0.0, 2.0 ** -149, 1 - 2.0 ** -24, 1.0, -1.0, float("nan")], device=cuda)
    got = ops.sample_tokens(x, last, 1.0, 17, 1.0, 0.0).tolist()
    order = torch.argsort(-x.float(), dim=1, stable=True).tolist()
    assert got == [order[0][0], order[1][0], order[2][16], order[3][16], order[4][0], order[5][0]]
    # over everything: with u near 1 the last token of positive weight
    y = torch.full((1, 500), -60.0, device=cuda)
    y[0, 3], y[0, 400], y[0, 499] = 0.0, -20.0, float("-inf")
    assert ops.sample_tokens(y, last[2:3])[0] == 3
    assert ops.sample_tokens(y, torch.ones(1, device=cuda))[0] == 400  # -60 is below 2^-45


def test_rows_that_are_not_finite(cuda):
    x = torch.randn(9, 20000, device=cuda)
    x[0, 700] = x[0, 900] = float("nan")
    x[1, 800] = x[1, 19000] = float("inf")
    x[2] = float("-inf")
    x[3] = float("-inf")
    x[3, 12345] = -7.0
    x[4, 17:] = float("-inf")
    x[5, ::2] = float("-inf")
    x[6, 0] = float("nan")
    x[6, 1] = float("inf")
    x[7] = 65504.0
    x[8] = -65504.0
    x[8, 5] = 65504.0
    u = torch.rand(9, device=cuda)
    for lg in (x, x.half()):
        for s in SETTINGS:
            check(lg, u, *s, close_allowed=1)
        got = ops.sample_tokens(lg, u, 1.5, 0, 0.9).tolist()
        assert got[0] == 700 and got[1] == 800 and got[2] == 0 and got[3] == 12345 and got[4] < 17 and got[5] % 2
        assert got[6] == 0 and got[8] == 5


def test_extreme_temperatures(cuda):
    x, u = rows(cuda, 4, 9000, 3)
    first = torch.argmax(x.float(), 1).tolist()
    for T in (1e-45, 1e-20):
        assert ops.sample_tokens(x, u, T).tolist() == first
    x[:, 8000:] = float("-inf")
    got = ops.sample_tokens(x, u, torch.full((4,), float("inf"), device=cuda))  # uniform over the finite ones, in order
    order = torch.argsort(-x.float(), dim=1, stable=True)
    assert got.tolist() == [int(order[b, int(u[b].double().item() * 8000)]) for b in range(4)]
    first = torch.argmax(x.float(), 1).tolist()  # without the masked ones
    assert ops.sample_tokens(x, u, torch.full((4,), float("nan"), device=cuda)).tolist() == first


def test_a_row_does_not_depend_on_the_batch(cuda):
    x, u = rows(cuda, 40, 33000, 8)
    for s in SETTINGS:
        whole = ops.sample_tokens(x, u, *s)
        one = torch.cat([ops.sample_tokens(x[b:b + 1], u[b:b + 1], *s) for b in range(0, 40, 7)])
        assert torch.equal(whole[::7], one)


def test_frequencies(cuda):
    """Tokens over evenly spread u come as often as their probabilities say, to one in n."""
    n = 4096
    l = torch.tensor([[0.0, 1.0, -2.0, 1.0, 0.5, float("-inf")]], device=cuda)
    u = (torch.arange(n, device=cuda) + 0.5) / n
    got = ops.sample_tokens(l.expand(n, 6).contiguous(), u.float(), 0.8)
    want = torch.softmax(l[0].double() / 0.8, 0) * n
    assert (torch.bincount(got.long(), minlength=6) - want).abs().max() <= 1


def test_strided_rows_outputs_and_workspaces(cuda):
    wide, u = rows(cuda, 5, 4001, 4)
    view = wide[:, 3:3800]
    want = ops.sample_tokens(view.contiguous(), u, 0.9, 30, 0.9)
    assert torch.equal(ops.sample_tokens(view, u, 0.9, 30, 0.9), want)
    ws = torch.full((_C.sample_tokens_workspace_bytes(5, 3797),), 255, dtype=torch.uint8, device=cuda)
    out = torch.full((5,), -1, dtype=torch.int32, device=cuda)
    assert ops.sample_tokens(view, u, 0.9, 30, 0.9, out=out, workspace=ws) is not None
    assert torch.equal(out, want)
    one = wide.as_strided((1, 4001), (0, 1))
    assert torch.equal(ops.sample_tokens(one, u[:1]), ops.sample_tokens(wide[:1], u[:1]))
    assert ops.sample_tokens(wide[:0], u[:0]).shape == (0,)


def test_largest_vocabulary(cuda):
    x, u = rows(cuda, 2, 524288, 6, spread=1.0, half=False)
    for s in SETTINGS[:6]:
        check(x, u, *s, close_allowed=1)
    with pytest.raises(RuntimeError, match="524288"):
        ops.sample_tokens(torch.zeros(1, 524289, device=cuda), u[:1])


def test_streams_and_graphs(cuda):
    x, u = rows(cuda, 30, 50000, 10)
    T = torch.full((30,), 0.9, device=cuda)
    k = torch.full((30,), 40, dtype=torch.int32, device=cuda)
    k[::3] = 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample_tokens(x, u, T, k, 0.9)
    side.synchronize()
    assert torch.equal(got, ops.sample_tokens(x, u, T, k, 0.9))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_tokens(x, u, T, k, 0.9)
    for i in range(4):
        y, v = rows(cuda, 30, 50000, 20 + i)
        x.copy_(y)
        u.copy_(v)
        T.fill_(0.0 if i == 2 else 0.5 + 0.3 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.sample_tokens(x, u, T, k, 0.9))


def test_refusals(cuda):
    x, u = rows(cuda, 3, 100, 1)
    k = torch.zeros(3, dtype=torch.int32, device=cuda)
    ws = torch.empty(64, dtype=torch.uint8, device=cuda)
    bad = [
        lambda: ops.sample_tokens(x.bfloat16(), u), lambda: ops.sample_tokens(x[0], u), lambda: ops.sample_tokens(x.t(), u),
        lambda: ops.sample_tokens(x[:1].expand(3, 100), u), lambda: ops.sample_tokens(x.cpu(), u),
        lambda: ops.sample_tokens(x, u[:2]), lambda: ops.sample_tokens(x, u.double()), lambda: ops.sample_tokens(x, u.cpu()),
        lambda: ops.sample_tokens(x, u, -1.0), lambda: ops.sample_tokens(x, u, float("nan")),
        lambda: ops.sample_tokens(x, u, 1.0, -1), lambda: ops.sample_tokens(x, u, 1.0, 0, 0.0),
        lambda: ops.sample_tokens(x, u, 1.0, 0, 1.1), lambda: ops.sample_tokens(x, u, 1.0, 0, 1.0, -0.1),
        lambda: ops.sample_tokens(x, u, 1.0, 0, 1.0, 1.1), lambda: ops.sample_tokens(x, u, u[:2]),
        lambda: ops.sample_tokens(x, u, k), lambda: ops.sample_tokens(x, u, 1.0, k.long()),
        lambda: ops.sample_tokens(x, u, out=k.long()), lambda: ops.sample_tokens(x, u, out=k[:2]),
        lambda: ops.sample_tokens(x, u, workspace=ws), lambda: ops.sample_tokens(x[:, :0], u),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was taken")


def test_outputs_over_an_input_are_refused(cuda):
    x, u = rows(cuda, 3, 100, 1)
    k = torch.zeros(3, dtype=torch.int32, device=cuda)
    f = torch.ones(3, device=cuda)
    i32 = torch.int32
    bad = [
        lambda: ops.sample_tokens(x, u, out=u.view(i32)), lambda: ops.sample_tokens(x, u, 1.0, k, out=k),
        lambda: ops.sample_tokens(x, u, f, out=f.view(i32)), lambda: ops.sample_tokens(x, u, 1.0, 0, f, out=f.view(i32)),
        lambda: ops.sample_tokens(x, u, 1.0, 0, 1.0, f, out=f.view(i32)),
    ]
    for i, g in enumerate(bad):
        with pytest.raises(RuntimeError, match="overlap"):
            g()
            pytest.fail(f"call {i} was taken")


@pytest.mark.parametrize("half", [True, False])
def test_numbers_of_collected_tokens(cuda, half):
    """Top-k up to 2048 collects about k tokens: numbers about the sizes that one wave, the workgroup with one or two tokens a
    thread, and the search take. Row b of the last logits has so many equal ones, which top-k cuts in their middle."""
    ks = [1, 2, 255, 256, 257, 300, 700, 1000, 1023, 1024, 1025, 1400, 1999, 2047, 2048]
    k = torch.tensor(ks, dtype=torch.int32, device=cuda)
    for i, (T, p, m) in enumerate([(1.0, 1.0, 0.0), (1.4, 0.9, 0.0), (0.9, 1.0, 0.01), (2.0, 0.97, 0.03), (5.0, 0.5, 1e-3)]):
        x, u = rows(cuda, len(ks), 30011, 40 + i, half=half)
        check(x, u, T, k, p, m)
    for n in (200, 256, 257, 1000, 1024, 1025, 2000, 2048, 2049, 4000, 4096, 4097):
        x, u = rows(cuda, len(ks), 9001, n, spread=0.5, half=half)
        x[:, 17:17 + n] = 30.0
        check(x, u, 1.0, k, 0.7, 0.0, close_allowed=1)
        check(x, u, 0.5, 0, 0.35, 0.5, close_allowed=1)
