"""Argument checks of soi_sample_tokens and soi_kv4_shared_attention: refused before any launch; their workspace queries."""
import ctypes as C

import pytest

from test_kv4_cpu import BAD_CACHES, LIB, cache

I, P, F, Z = C.c_int64, C.c_void_p, C.c_float, C.c_size_t
A = 1 << 20  # an address, never read


@pytest.fixture(scope="module")
def lib():
    import torch  # noqa: F401

    L = C.CDLL(str(LIB))
    L.soi_last_error.restype = C.c_char_p
    L.soi_sample_tokens_workspace_bytes.argtypes = [I] * 2
    L.soi_sample_tokens_workspace_bytes.restype = Z
    L.soi_sample_tokens.argtypes = [P, C.c_int, I, I, I, P, P, F, P, C.c_int32, P, F, P, F, P, P, Z, P]
    L.soi_kv4_shared_attention_workspace_bytes.argtypes = [I] * 7
    L.soi_kv4_shared_attention_workspace_bytes.restype = Z
    L.soi_kv4_shared_attention.argtypes = [P, P, I, I, P, I, P, I, I, P, F, P, Z, P]
    return L


def sample(lib, **change):
    a = dict(logits=A, f32=0, stride=1000, B=2, V=1000, u=A, T=None, T_all=1.0, k=None, k_all=0, p=None, p_all=1.0, m=None,
             m_all=0.0, tokens=A, ws=A, ws_bytes=1 << 40, stream=None) | change
    return lib.soi_sample_tokens(*a.values())


@pytest.mark.parametrize("change,text", [
    (dict(B=-1), b"rows"), (dict(B=65536), b"rows"), (dict(V=0), b"logits"), (dict(V=524289, stride=524289), b"logits"),
    (dict(stride=999), b"overlap"), (dict(stride=-1), b"overlap"), (dict(logits=None), b"null"), (dict(u=None), b"null"),
    (dict(tokens=None), b"null")])
def test_sample_refusals(lib, change, text):
    assert sample(lib, **change) == 1
    assert text in lib.soi_last_error()


def test_sample_workspace(lib):
    need = lib.soi_sample_tokens_workspace_bytes(2, 1000)
    for change in (dict(ws=None), dict(ws=A + 8), dict(ws_bytes=need - 1)):
        assert sample(lib, **change) == 2
        assert b"workspace" in lib.soi_last_error()
    for B, V in ((0, 10), (-1, 10), (65536, 10), (1, 0), (1, 524289)):
        assert lib.soi_sample_tokens_workspace_bytes(B, V) == 0
    assert sample(lib, B=0, logits=None, u=None, tokens=None, ws=None, ws_bytes=0) == 0
    # no number of rows makes another number of them need less
    sizes = [lib.soi_sample_tokens_workspace_bytes(b, 524288) / b for b in (1, 2, 16, 1024, 65535)]
    assert min(sizes) > 32768 and max(sizes) < 50000


def shared(lib, c=None, **change):
    a = dict(q=0x7000, q_stride=4 * 128, NQ=4, cu=A, groups=1, lens=A, max_len=256, max_shared=128, out=0x8000, scale=0.1, ws=A,
             ws_bytes=1 << 40, stream=None) | change
    return lib.soi_kv4_shared_attention(C.byref(c if c is not None else cache()), *a.values())


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_shared_caches(lib, bad):
    assert shared(lib, cache(**bad)) == 1


@pytest.mark.parametrize("change,text", [
    (dict(NQ=0), b"num_q_heads"), (dict(NQ=3), b"num_q_heads"), (dict(NQ=65536), b"num_q_heads"), (dict(groups=-1), b"groups"),
    (dict(groups=2049), b"groups"), (dict(q_stride=511), b"overlap"), (dict(max_len=-1), b"max_len"), (dict(max_len=257), b"max_len"),
    (dict(max_shared=-1), b"max_shared"), (dict(max_shared=257), b"max_shared"), (dict(max_len=64, max_shared=65), b"max_shared"),
    (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"), (dict(scale=float("inf")), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(cu=None), b"null"),
    (dict(lens=None), b"null"), (dict(out=0x7000), b"out = q")])
def test_shared_refusals(lib, change, text):
    assert shared(lib, **change) == 1
    assert text in lib.soi_last_error()


def test_shared_sequences_and_workspace(lib):
    assert shared(lib, cache(batch=2049)) == 1 and b"2048" in lib.soi_last_error()
    need = lib.soi_kv4_shared_attention_workspace_bytes(2, 1, 4, 2, 128, 256, 128)
    assert need > 0
    for change in (dict(ws=None), dict(ws=A + 8), dict(ws_bytes=need - 1)):
        assert shared(lib, **change) == 2
        assert b"workspace" in lib.soi_last_error()
    for bad in ((0, 1, 4, 2, 128, 256, 128), (2049, 1, 4, 2, 128, 256, 128), (2, -1, 4, 2, 128, 256, 128), (2, 1, 3, 2, 128, 256, 128),
                (2, 1, 4, 0, 128, 256, 128), (2, 1, 4, 2, 0, 256, 128), (2, 1, 4, 2, 128, -1, 0), (2, 1, 4, 2, 128, 256, 257)):
        assert lib.soi_kv4_shared_attention_workspace_bytes(*bad) == 0
