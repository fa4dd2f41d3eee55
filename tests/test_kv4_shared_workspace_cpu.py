"""How large a workspace attention over shared pages asks for: a state for each column and each unit more than there are tiles."""
import pytest

from test_sample_kv4_shared_cpu import lib  # noqa: F401


@pytest.mark.parametrize("B,G,NQ,NKV,hd,length,shared,most", [
    (2048, 1024, 32, 8, 128, 4096, 4096, 85e6), (2048, 2048, 64, 8, 128, 4096, 4096, 160e6), (64, 1, 32, 8, 128, 8704, 8192, 45e6),
    (1, 1, 1, 1, 64, 64, 0, 1e4)])
def test_size(lib, B, G, NQ, NKV, hd, length, shared, most):  # noqa: F811
    states = 2 * B * NQ * (hd + 4) * 4  # of each (sequence, head): one over the shared tokens, one over the others
    assert 0 < lib.soi_kv4_shared_attention_workspace_bytes(B, G, NQ, NKV, hd, length, shared) <= most
    if shared:
        assert lib.soi_kv4_shared_attention_workspace_bytes(B, G, NQ, NKV, hd, length, shared) >= states
