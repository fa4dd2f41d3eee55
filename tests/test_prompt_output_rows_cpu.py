"""Prompt attention refuses an output whose rows share memory: two workgroups would write there, in any order. Argument checks
of the C entry, which come before any HIP call; what passes them stops at the workspace, which is not given."""
import pytest

from test_kv4_cpu import error, lib  # noqa: F401  (the fixture)

NQ, HD, TQ = 4, 128, 8


def call(lib, token_stride, head_stride, heads=NQ, tokens=TQ):  # noqa: F811
    st = lib.soi_prompt_attention(16, 512, 128, 32, 256, 128, 48, 256, 128, 64, 64, 1, tokens, 1 << 20, tokens, heads, 2, HD, 1024,
                                  token_stride, head_stride, 1.0, None, 0, None)
    return st, error(lib, st)


@pytest.mark.parametrize("ts,hs", [(0, 128), (0, 0), (512, 0), (512, 64), (256, 128), (64, 1024), (128, 512), (384, 256), (120, 8 * 128),
                                   (-512, 64), (-256, 128), (256, -128)])
def test_shared_rows(lib, ts, hs):  # noqa: F811
    st, text = call(lib, ts, hs)
    assert st == 1 and "overlap" in text


@pytest.mark.parametrize("ts,hs", [(512, 128), (4096, 128), (128, 8 * 128), (132, 1200), (1024, 256), (-512, 128), (512, -128),
                                   (128, -1024), (5 * 128, 2 * 128), (3 * 128, 9 * 3 * 128)])
def test_rows_of_their_own(lib, ts, hs):  # noqa: F811
    st, text = call(lib, ts, hs)
    assert st == 2 and "workspace" in text


def test_strides_that_nothing_is_multiplied_by(lib):  # noqa: F811
    """One token, or one head: its stride says nothing."""
    for ts, hs, heads, tokens in ((0, 128, 4, 1), (4, 128, 4, 1), (0, 0, 2, 1), (512, 0, 2, 1)):
        st, text = call(lib, ts, hs, heads, tokens)
        assert (st == 1) == (hs == 0), (ts, hs, text)


def test_against_a_count_of_the_elements(lib):  # noqa: F811
    rows = [(i, j) for i in range(TQ) for j in range(NQ)]
    for ts in range(-8, 9):
        for hs in range(-33, 34):
            at = [i * ts * 64 + j * hs * 64 for i, j in rows]
            shared = len({x // 64 + d for x in at for d in (0, 1)}) < 2 * len(rows)
            st, text = call(lib, ts * 64, hs * 64)
            assert (st == 1 and "overlap" in text) == shared, (ts, hs, text)
