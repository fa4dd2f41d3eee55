"""PagedKV4.fork: pages that sequences hold together, and the groups that a step finds among them."""
import pytest

from test_paged_kv import make


def test_forks_hold_whole_pages_together():
    c = make(num_pages=10, max_len=100)
    a = c.add()
    c.step({a: 40})                                       # pages of 16: two whole ones, one begun
    b = c.fork(a)
    d = c.fork(a, 31)
    assert (c.length(b), c.length(d), c.free_pages) == (32, 16, 7)
    s = c.step({a: 1, b: 1, d: 1})
    t = s.block_table.tolist()
    assert t[0][:2] == t[1][:2] and t[0][0] == t[2][0] and len({t[0][2], t[1][2], t[2][1]}) == 3
    assert c.free_pages == 5 and s.lens == (41, 33, 17)
    c.free(a)                                             # its own page only
    assert c.free_pages == 6
    e = c.fork(b, 32)
    c.free(b)
    assert c.free_pages == 7 and c.step({e: 0, d: 0}).block_table.tolist()[0][:2] == t[1][:2]
    c.free(e)
    assert c.free_pages == 8                              # the second page; d holds the first and its own
    c.free(d)
    assert c.free_pages == 10 and not c._users
    with pytest.raises(KeyError):
        c.fork(d)


def test_forks_of_nothing_and_refusals():
    c = make()
    a = c.add()
    b = c.fork(a)
    assert c.length(b) == 0
    c.step({a: 20})
    for bad in (-1, 21):
        with pytest.raises(ValueError, match="holds 20 tokens"):
            c.fork(a, bad)
    assert c.length(c.fork(a, 15)) == 0 and c.free_pages == 4


def groups(c, *seqs):
    s = c.step({x: 0 for x in seqs})
    return s.cu_groups is None or (s.cu_groups.tolist(), s.shared_lens.tolist(), s.max_shared)


def test_a_step_groups_neighbours():
    c = make(num_pages=60, max_len=400)
    a, z = c.add(), c.add()
    c.step({a: 100, z: 70})                               # six whole pages, four
    b, d, e, y = c.fork(a), c.fork(a, 90), c.fork(a, 20), c.fork(z)
    c.step({b: 5, d: 5, e: 5, y: 5})
    assert groups(c, a, b) == ([0, 2], [96, 96], 96)
    assert groups(c, a, b, d) == ([0, 3], [80] * 3, 80)   # 3 x 5 pages instead of 2 x 6
    assert groups(c, a, b, d, e) == ([0, 3, 4], [80, 80, 80, 0], 80)  # 4 x 1 page would read more
    assert groups(c, a, e) == ([0, 2], [16, 16], 16)
    assert groups(c, a, b, z, y) == ([0, 2, 4], [96, 96, 64, 64], 96)
    assert groups(c, z, a, y, b) is True                  # no neighbours share
    assert groups(c, a) is True
    f = c.add()
    assert groups(c, f, a, b) == ([0, 1, 3], [0, 96, 96], 96)
    assert groups(c, a, b, f) == ([0, 2, 3], [96, 96, 0], 96)


def test_without_forks_nothing_is_shared():
    c = make()
    a, b = c.add(), c.add()
    assert c.step({a: 30, b: 30}).cu_groups is None
    x = c.fork(a)
    c.free(x)
    assert c.step({a: 1, b: 1}).cu_groups is None
