"""Argument checks of the 8-bit row and product entry points: refused before any launch."""
import ctypes as C
from pathlib import Path

import pytest

LIB = Path(__file__).resolve().parent.parent / "sparse-offload-infer_amd" / "soinfer" / "libsoinfer_hip.so"
P, I, D = C.c_void_p, C.c_int64, C.c_double


@pytest.fixture(scope="module")
def lib():
    import torch  # noqa: F401

    L = C.CDLL(str(LIB))
    L.soi_last_error.restype = C.c_char_p
    L.soi_int8_rows.argtypes = [P, I, P, I, P, D, I, I, P, P, P, P]
    L.soi_int8_linear.argtypes = [P, P, P, P, P, P, I, I, I, P]
    L.soi_int8_gate_up.argtypes = [P, P, P, P, P, P, P, I, I, I, P]
    return L


A = 1 << 20  # an address, never read


@pytest.mark.parametrize("change,text", [
    (dict(H=24), b"multiple of 16"), (dict(H=0), b"multiple of 16"), (dict(H=65552), b"65536"), (dict(T=-1), b"rows"),
    (dict(T=1 << 22), b"rows"), (dict(sum=None), b"come together"), (dict(weight=None), b"norm weight"),
    (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps"), (dict(q=None), b"null"),
    (dict(x=None), b"null"), (dict(scale=None), b"null"), (dict(xs=63), b"overlap"), (dict(rs=0), b"overlap"),
    (dict(q=A + 8), b"aligned"), (dict(sum=A + 4), b"aligned")])
def test_rows(lib, change, text):
    a = dict(x=A, xs=64, res=A, rs=64, weight=A, eps=1e-6, T=2, H=64, q=A, scale=A, sum=A) | change
    assert lib.soi_int8_rows(*a.values(), None) == 1
    assert text in lib.soi_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(K=24), b"multiple of 16"), (dict(K=131072), b"131072"), (dict(K=0), b"multiple of 16"), (dict(N=0), b"outputs"),
    (dict(T=-1), b"outputs"), (dict(T=1 << 22), b"outputs"), (dict(N=1 << 22), b"outputs"), (dict(x=None), b"null"),
    (dict(sx=None), b"null"), (dict(w=None), b"null"), (dict(sw=None), b"null"), (dict(y=None), b"null"),
    (dict(x=A + 8), b"aligned"), (dict(w=A + 4), b"aligned")])
def test_products(lib, change, text):
    a = dict(x=A, sx=A, w=A, sw=A, y=A, T=2, N=8, K=64) | change
    assert lib.soi_int8_linear(a["x"], a["sx"], a["w"], a["sw"], None, a["y"], a["T"], a["N"], a["K"], None) == 1
    assert text in lib.soi_last_error()
    for order in ((a["w"], a["sw"], A, A), (A, A, a["w"], a["sw"])):
        assert lib.soi_int8_gate_up(a["x"], a["sx"], *order, a["y"], a["T"], a["N"], a["K"], None) == 1
        assert text in lib.soi_last_error()


def test_no_rows_need_no_pointers(lib):
    assert lib.soi_int8_rows(None, 0, None, 0, None, 0.0, 0, 64, None, None, None, None) == 0
    assert lib.soi_int8_linear(None, None, None, None, None, None, 0, 8, 64, None) == 0
    assert lib.soi_int8_gate_up(None, None, None, None, None, None, None, 0, 8, 64, None) == 0
