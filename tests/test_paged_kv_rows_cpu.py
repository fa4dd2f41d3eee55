"""PagedKV4 refuses rows and tables that do not cover a step: its tokens count as cached once the step is made, and what
nobody wrote would be read from the pages' earlier sequence."""
import pytest
import torch

from soinfer import ops
from soinfer.runtime.paged_kv import PagedKV4

NQ, NKV, HD = 4, 2, 64


@pytest.fixture
def cache(monkeypatch):
    """A cache whose operators only say that they were called."""
    for name in ("kv4_append", "kv4_decode_attention", "prompt_attention"):
        monkeypatch.setattr(ops, name, lambda *a, name=name, **k: name)
    return PagedKV4(1, 12, NKV, HD, max_len=100, group_size=32, page_size=16, device="cpu")


def rows(n, heads=NQ + 2 * NKV):
    return torch.zeros((n, heads * HD), dtype=torch.float16)


def tables(n, m=None):
    return torch.zeros((n, HD // 2)), torch.zeros((n if m is None else m, HD // 2))


def test_append_needs_every_row_of_the_step(cache):
    a, b = cache.add(), cache.add()
    step = cache.step({a: 5, b: 3})
    assert cache.append(0, step, rows(8), None, None, *tables(100), NQ) == "kv4_append"
    assert cache.append(0, step, rows(11), None, None, *tables(100), NQ) == "kv4_append"  # rows behind the last sequence
    for n in (0, 7):
        with pytest.raises(ValueError, match="8 rows"):
            cache.append(0, step, rows(n), None, None, *tables(100), NQ)


def test_append_needs_every_position_in_the_tables(cache):
    a, b = cache.add(), cache.add()
    cache.step({a: 40})
    step = cache.step({a: 0, b: 30})  # a's 40 positions are not turned again
    assert cache.append(0, step, rows(30), None, None, *tables(30), NQ) == "kv4_append"
    for t in (tables(29), tables(30, 29), tables(29, 30)):
        with pytest.raises(ValueError, match="30 positions"):
            cache.append(0, step, rows(30), None, None, *t, NQ)
    step = cache.step({a: 1})
    with pytest.raises(ValueError, match="41 positions"):
        cache.append(0, step, rows(1), None, None, *tables(40), NQ)


def test_prompt_needs_every_row_of_the_step(cache):
    a = cache.add()
    step = cache.step({a: 5})
    q, k, v = (torch.zeros((5, h, HD), dtype=torch.float16) for h in (NQ, NKV, NKV))
    assert cache.prompt(0, step, q, k, v) == "prompt_attention"
    for bad in ((q[:4], k, v), (q, k[:4], v), (q, k, v[:4])):
        with pytest.raises(ValueError, match="5 rows"):
            cache.prompt(0, step, *bad)


def test_rows_of_a_context_are_named_first(cache):
    """k and v of the new rows for a sequence that had some already: that is the mistake, however many rows there are."""
    a = cache.add()
    cache.step({a: 5})
    step = cache.step({a: 3})
    q, k, v = (torch.zeros((2, h, HD), dtype=torch.float16) for h in (NQ, NKV, NKV))
    with pytest.raises(ValueError, match="begin"):
        cache.prompt(0, step, q, k, v)
