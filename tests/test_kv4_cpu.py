"""The paged 4-bit cache and prompt attention without a GPU: argument checks of the C ABI (they come before any HIP call),
the workspace query, and the reference's own byte layout."""
import ctypes as C
from pathlib import Path

import numpy as np
import pytest

import kv4_ref as R

LIB = Path(__file__).resolve().parent.parent / "sparse-offload-infer_amd" / "soinfer" / "libsoinfer_hip.so"


class CacheArg(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k_pages", "k_scale", "v_pages", "v_scale", "block_table", "seq_lens")] + \
        [(n, C.c_int64) for n in ("batch", "max_blocks", "num_pages", "num_kv_heads", "page_size", "head_dim", "group_size")]


@pytest.fixture(scope="module")
def lib():
    import torch  # noqa: F401  (same HIP runtime as the product process)

    lib = C.CDLL(str(LIB))
    lib.soi_last_error.restype = C.c_char_p
    i, p, f = C.c_int64, C.c_void_p, C.c_float
    lib.soi_kv4_append.argtypes = [p, p, i, p, p, p, p, i, p, i, i, p, p, f, p]
    lib.soi_kv4_read.argtypes = [p, p, i, p, p, p]
    lib.soi_kv4_decode_attention.argtypes = [p, p, i, i, i, p, f, p, C.c_size_t, p]
    lib.soi_kv4_decode_attention_workspace_bytes.argtypes = [i] * 5
    lib.soi_kv4_decode_attention_workspace_bytes.restype = C.c_size_t
    lib.soi_prompt_attention.argtypes = [p, i, i, p, i, i, p, i, i, p, p, i, i, i, i, i, i, i, p, i, i, f, p, C.c_size_t, p]
    lib.soi_prompt_attention_workspace_bytes.argtypes = [i] * 4
    lib.soi_prompt_attention_workspace_bytes.restype = C.c_size_t
    return lib


def cache(**change):
    at = dict(k_pages=0x1000, k_scale=0x2000, v_pages=0x3000, v_scale=0x4000, block_table=0x5000, seq_lens=0x6000, batch=2,
              max_blocks=4, num_pages=8, num_kv_heads=2, page_size=64, head_dim=128, group_size=64) | change
    return CacheArg(**at)


BAD_CACHES = [dict(head_dim=96), dict(head_dim=32), dict(group_size=16), dict(group_size=128, head_dim=64), dict(page_size=8),
              dict(page_size=48), dict(page_size=0), dict(num_pages=0), dict(num_pages=1 << 31), dict(num_kv_heads=0),
              dict(batch=0), dict(batch=65536), dict(max_blocks=0), dict(max_blocks=1 << 25), dict(k_pages=None),
              dict(v_scale=None), dict(block_table=None), dict(seq_lens=None), dict(k_pages=0x1008), dict(k_scale=0x2002)]


def error(lib, status):
    assert status in (1, 2, 4)
    return lib.soi_last_error().decode()


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_cache_checks(lib, bad):
    c = C.byref(cache(**bad))
    assert "soi_kv4_append" in error(lib, lib.soi_kv4_append(c, 1, 8 * 128, None, None, 16, 16, 4, 16, 2, 4, 16, None, 1e-6, None))
    assert "soi_kv4_read" in error(lib, lib.soi_kv4_read(c, 16, 2, 16, 32, None))
    assert "soi_kv4_decode_attention" in error(lib, lib.soi_kv4_decode_attention(c, 16, 512, 4, 64, 32, 1.0, None, 0, None))


def test_call_checks(lib):
    c = C.byref(cache())
    ok = [c, 16, 8 * 128, None, None, 16, 16, 4, 16, 2, 4, 16, None, 1e-6, None]
    for at, bad, text in ((2, 8 * 128 - 1, "overlap"), (3, 16, "together"), (7, 0, "table"), (8, None, "null"), (9, -1, "token"),
                          (10, 0, "num_q_heads"), (11, None, "null"), (11, 24, "aligned"), (12, 24, "aligned")):
        args = list(ok)
        args[at] = bad
        assert text in error(lib, lib.soi_kv4_append(*args))
    assert lib.soi_kv4_append(*ok[:9], 0, *ok[10:]) == 0  # no tokens: nothing to do
    assert lib.soi_kv4_read(c, 16, 0, None, None, None) == 0
    assert "k_out = v_out" in error(lib, lib.soi_kv4_read(c, 16, 2, 16, 16, None))
    assert "token" in error(lib, lib.soi_kv4_read(c, 16, -2, 16, 32, None))
    ok = [c, 16, 4 * 128, 4, 256, 32, 1.0, None, 0, None]
    for at, bad, text in ((2, 4 * 128 - 8, "overlap"), (3, 3, "multiple"), (3, 0, "multiple"), (4, 257, "max_len"),
                          (4, -1, "max_len"), (5, 16, "out = q"), (6, 0.0, "scale"), (6, float("nan"), "scale")):
        args = list(ok)
        args[at] = bad
        assert text in error(lib, lib.soi_kv4_decode_attention(*args))
    long = C.byref(cache(max_blocks=100))
    st = lib.soi_kv4_decode_attention(long, 16, 512, 4, 6400, 32, 1.0, None, 0, None)
    assert st == 2 and "workspace" in error(lib, st)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_more_tokens_than_one_launch(lib, hd):
    """512 / hd tokens a workgroup of 256, and a grid holds fewer than 2^32 work items."""
    c = C.byref(cache(head_dim=hd, group_size=32))
    T = ((1 << 24) - 1) * (512 // hd) + 1
    assert "tokens" in error(lib, lib.soi_kv4_append(c, 16, 8 * hd, None, None, 16, 16, 4, 16, T, 4, 16, None, 1e-6, None))
    assert "tokens" in error(lib, lib.soi_kv4_read(c, 16, T, 16, 32, None))


def test_workspace_query(lib):
    q = lib.soi_kv4_decode_attention_workspace_bytes
    assert q(1, 4, 2, 128, 64) == 0 and q(1, 4, 2, 128, 0) == 0  # one split: none
    n = q(1, 4, 2, 128, 4096)
    assert n > 0 and n % (4 * 130 * 4) == 0
    assert q(0, 4, 2, 128, 64) == 0 and q(1, 3, 2, 128, 4096) == 0 and q(1, 4, 2, 128, -1) == 0


def test_prompt_attention_checks(lib):
    # q, 3 x (pointer, token stride, head stride), cu_q, cu_k, batch, Tq, Tk, max_q, NQ, NKV, hd, out, strides, scale, workspace, its bytes, stream
    ok = [16, 512, 128, 32, 256, 128, 48, 256, 128, 64, 64, 1, 8, 8, 8, 4, 2, 128, 1024, 512, 128, 1.0, None, 0, None]
    for at, bad, text in ((17, 100, "multiple of 8"), (17, 264, "up to 256"), (17, 0, "head_dim"), (15, 3, "multiple of num_kv"),
                          (15, 0, "multiple"), (11, 0, "sequences"), (11, 65536, "sequences"), (12, -1, "token"),
                          (13, 1 << 30, "token"), (14, -1, "max_q"), (21, 0.0, "scale"), (21, float("inf"), "scale"),
                          (0, None, "null"), (3, None, "null"), (9, None, "null"), (18, None, "null"), (3, 40, "aligned"),
                          (4, 260, "aligned"), (8, 132, "aligned"), (18, 1028, "8-byte"), (20, 126, "8-byte")):
        args = list(ok)
        args[at] = bad
        assert text in error(lib, lib.soi_prompt_attention(*args)), (at, bad)
    args = list(ok)
    args[13] = 8192  # 8 queries over 8192 keys: split
    st = lib.soi_prompt_attention(*args)
    assert st == 2 and "workspace" in error(lib, st)
    assert lib.soi_prompt_attention(*ok[:12], 0, *ok[13:]) == 0
    assert lib.soi_prompt_attention(*ok[:14], 0, *ok[15:]) == 0


@pytest.mark.parametrize("at", [1, 4, 7])
def test_prompt_rows_too_far_apart(lib, at):
    """128 rows of a tile, and the bytes behind the first, have to fit a 32-bit offset."""
    args = [16, 512, 128, 32, 256, 128, 48, 256, 128, 64, 64, 1, 8, 8, 8, 4, 2, 128, 1024, 512, 128, 1.0, None, 0, None]
    args[at] = 1 << 22
    assert "apart" in error(lib, lib.soi_prompt_attention(*args))


def test_prompt_workspace_query(lib):
    q = lib.soi_prompt_attention_workspace_bytes
    assert q(8, 100, 4, 128) == 0 and q(0, 4096, 4, 128) == 0 and q(1 << 16, 1 << 16, 16, 128) == 0
    n = q(8, 8192, 4, 128)
    assert n > 0 and n % (8 * 4 * 130 * 4) == 0
    for rows in (1, 100, 1000, 8000):  # bounded whatever the rows: at most about 2^16 of them with the splits counted
        for heads in (1, 8, 64):
            assert q(rows, 1 << 20, heads, 256) <= 2 * 65536 * 258 * 4


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_reference_layout_is_a_permutation(hd):
    """Every dimension has one nibble of its token, in K's words and in V's units."""
    seen_k, seen_v = set(), set()
    for d in range(hd):
        q = np.zeros(hd, np.int8)
        q[d] = 1
        k = R.k_row_bytes(q)
        assert np.count_nonzero(k) == 1
        seen_k.add((int(np.flatnonzero(k)[0]), int(k.max())))
        v = {a: x for a, x in R.v_row_units(q).items() if x}
        assert len(v) == 1
        seen_v.add(next(iter(v.items())))
    assert len(seen_k) == len(seen_v) == hd


def test_reference_quantizer():
    x = np.array([7, 0.5, 1.5, 2.5, -0.5, -7] + [0] * 26, np.float16)
    q, s = R.quantize(x, 32)
    assert s[0] == 1 and q[:6].tolist() == [7, 0, 2, 2, 0, -7]
    for bad in (np.inf, np.nan):
        x[3] = bad
        q, s = R.quantize(x, 32)
        assert not q.any() and not np.isfinite(s[0]) and np.isnan(R.values(q, s)).all()
