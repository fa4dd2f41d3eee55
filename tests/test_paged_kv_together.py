"""PagedKV4.attend takes the attention over shared pages where it is the faster one, and gives the same either way."""
import math

import pytest
import torch

import kv4_ref as R
from test_paged_kv import make


def taken(monkeypatch, c, step, NQ):
    """Which operator a decode step's attention calls."""
    from soinfer import ops

    calls = []
    for name in ("kv4_shared_attention", "kv4_decode_attention"):
        monkeypatch.setattr(ops, name, lambda *a, name=name, **k: calls.append(name))
    c.attend(0, step, torch.zeros(len(step.sequences), NQ, c.head_dim, dtype=torch.float16))
    assert len(calls) == 1
    return calls[0]


def forks(c, n, prompt, more):
    """A sequence of `prompt` tokens, n - 1 that begin with its pages, and `more` tokens for each."""
    a = c.add()
    c.step({a: prompt})
    return c.step({s: more for s in [a] + [c.fork(a) for _ in range(n - 1)]})


def test_many_sequences_of_one_long_prompt(monkeypatch):
    c = make(layers=1, num_pages=200, num_kv_heads=8, head_dim=128, group_size=64, page_size=64, max_len=9000)
    assert taken(monkeypatch, c, forks(c, 64, 8192, 1), 32) == "kv4_shared_attention"


def test_a_shared_page_among_long_contexts_of_their_own(monkeypatch):
    c = make(layers=1, num_pages=6100, num_kv_heads=8, head_dim=64, max_len=2100)
    a = c.add()
    c.step({a: 16})
    step = c.step({s: 2000 for s in [a, c.fork(a)] + [c.add() for _ in range(46)]})
    assert step.groups == ((2, 16),) + ((1, 0),) * 46
    assert taken(monkeypatch, c, step, 32) == "kv4_decode_attention"


@pytest.mark.parametrize("n,prompt,more", [(2, 16, 1), (6, 500, 100), (48, 48, 1), (10, 1024, 1)])
def test_little_that_is_shared(monkeypatch, n, prompt, more):
    c = make(layers=1, num_pages=1200, num_kv_heads=2, head_dim=64, max_len=1200)
    assert taken(monkeypatch, c, forks(c, n, prompt, more), 4) == "kv4_decode_attention"


def test_heads_of_256(monkeypatch):
    c = make(layers=1, num_pages=200, num_kv_heads=2, head_dim=256, group_size=64, page_size=64, max_len=9000)
    assert taken(monkeypatch, c, forks(c, 64, 8192, 1), 16) == "kv4_decode_attention"


def test_a_step_without_forks(monkeypatch):
    c = make()
    a = c.add()
    assert taken(monkeypatch, c, c.step({a: 5}), 4) == "kv4_decode_attention"


@pytest.mark.gpu
@pytest.mark.parametrize("n,prompt,together", [(48, 4096, True), (40, 4096, False), (3, 100, False)])  # (519104 and 388896 of 400000)
def test_the_same_either_way(cuda, n, prompt, together):
    from soinfer import ops

    NQ, NKV, hd, gs = 16, 4, 128, 64
    c = make(layers=1, num_pages=160, num_kv_heads=NKV, head_dim=hd, group_size=gs, page_size=64, max_len=4200, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(n)
    rows = lambda t: torch.randn(t, NQ + 2 * NKV, hd, generator=g, device=cuda).half().flatten(1)  # noqa: E731
    cos, sin = (torch.from_numpy(x).to(cuda) for x in R.rope_tables(4200, hd))
    a = c.add()
    c.append(0, c.step({a: prompt}), rows(prompt), None, None, cos, sin, NQ)
    step = c.step({s: 9 for s in [a] + [c.fork(a) for _ in range(n - 1)]})
    c.append(0, step, rows(step.tokens), None, None, cos, sin, NQ)
    q = torch.randn(n, NQ, hd, generator=g, device=cuda).half()
    assert c._together(step, NQ) is together
    got, other = c.attend(0, step, q), ops.kv4_decode_attention(q, *c._layer(0), step.block_table, step.seq_lens, step.max_len)
    k, v, cu = c.read(0, step)
    for b, ln in enumerate(step.lens):
        kb, vb = (x[int(cu[b]):int(cu[b]) + ln].double() for x in (k, v))
        last = torch.full((1,), ln - 1, device=cuda)
        ref, bound = R.attention(q[b:b + 1].double(), kb, vb, last, 1 / math.sqrt(hd))
        # read rounds K and V to binary16 (u): a score by u sum |q k| scale at most, a value by u
        d = (q[b].double().abs() @ kb.abs().amax((0, 1))).amax() / math.sqrt(hd) * R.U
        wide = bound + (2 * d + 2 * R.U) * vb.abs().amax()
        R.assert_within(got[b:b + 1], ref, wide, f"sequence {b}")
        R.assert_within(other[b:b + 1], ref, wide, f"sequence {b}, decode")


def test_the_choice_is_made_once_a_step(monkeypatch):
    """Every layer of a step attends alike, and the rule's loop over the groups runs for the first of them."""
    from soinfer import ops

    c = make(layers=3, num_pages=60, num_kv_heads=2, head_dim=64, max_len=400)
    step = forks(c, 5, 64, 1)
    made = []
    monkeypatch.setattr(c, "_together", lambda s, n: made.append(n) or n == 4)
    calls = []
    for name in ("kv4_shared_attention", "kv4_decode_attention"):
        monkeypatch.setattr(ops, name, lambda *a, name=name, **k: calls.append(name))
    for heads in (4, 4, 8, 4):
        c.attend(0, step, torch.zeros(5, heads, 64, dtype=torch.float16))
    assert made == [4, 8] and calls == ["kv4_shared_attention"] * 2 + ["kv4_decode_attention", "kv4_shared_attention"]
