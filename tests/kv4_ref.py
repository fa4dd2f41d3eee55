"""Plain 64-bit references of the paged 4-bit KV cache and of packed prompt attention, for the tests.

The cache format is restated here nibble by nibble in numpy (include/soinfer_amd.h), apart from the kernels.

Tolerances, from the kernels' roundings (u = 2^-11 is half a binary16 step, relative; e = 2^-24 half a binary32 step):
  * an output is one binary16 rounding: u |ref| (2^-25 below the normal range);
  * the weights of V are rounded to binary16 before the product: u A, A = sum p |v| / sum p, and 2^-25 each where they
    are below the normal range;
  * a score's error d moves its weight by d, relatively: 2 d A, with d = (n + 8) e sum |q k| scale for n binary32
    additions of exact products and a few roundings, and 2^-21 for the exponential;
  * sums of n terms in binary32: n e A (the sum of p enters the same way: twice).
"""
from __future__ import annotations

import numpy as np
import torch

AWQ = (0, 2, 4, 6, 1, 3, 5, 7)
U, E, TINY = 2.0 ** -11, 2.0 ** -24, 2.0 ** -25


def quantize(x: np.ndarray, gs: int):
    """x fp16 [..., hd] -> codes int8 [..., hd], scales fp16 [..., hd / gs] (ties to even, codes 0 where the scale is not
    a positive number)."""
    g = x.astype(np.float64).reshape(*x.shape[:-1], -1, gs)
    with np.errstate(invalid="ignore", over="ignore"):
        s = (np.abs(g).max(-1) / 7).astype(np.float16)
    live = np.isfinite(s) & (s > 0)
    div = np.where(live, s, 1).astype(np.float64)[..., None]
    q = np.where(live[..., None], np.clip(np.rint(np.where(np.isfinite(g), g, 0) / div), -7, 7), 0)
    return q.reshape(x.shape).astype(np.int8), s


def values(q: np.ndarray, s: np.ndarray) -> np.ndarray:
    gs = q.shape[-1] // s.shape[-1]
    with np.errstate(invalid="ignore"):
        return q.astype(np.float64) * np.repeat(s.astype(np.float64), gs, -1)


def k_row_bytes(q: np.ndarray) -> np.ndarray:
    """codes [hd] -> a token's k_pages bytes [hd / 2]."""
    hd = q.size
    w = hd // 32
    words = np.zeros(hd // 8, np.uint32)
    for g in range(4):
        for i in range(w):
            for n in range(8):
                words[w * g + i] |= np.uint32((int(q[8 * (4 * i + g) + AWQ[n]]) & 15) << (4 * n))
    return words.view(np.uint8)


def v_row_units(q: np.ndarray) -> dict:
    """codes [hd] -> {(m, u): 16-bit unit}."""
    return {(m, u): sum((int(q[64 * u + 16 * n + m]) & 15) << (4 * n) for n in range(4))
            for m in range(16) for u in range(q.size // 64)}


class Cache:
    """Host image of the pages, written token by token."""

    def __init__(self, P, NKV, page, hd, gs, fill=0):
        self.P, self.NKV, self.page, self.hd, self.gs = P, NKV, page, hd, gs
        self.k = np.full((P, NKV, page, hd // 2), fill, np.uint8)
        self.v = np.full((P, NKV, page, hd // 2), fill, np.uint8)
        self.ks = np.zeros((P, NKV, hd // gs, page), np.float16)
        self.vs = np.zeros((P, NKV, hd // gs, page), np.float16)

    def put(self, pg, head, slot, k, v):
        """k, v fp16 [hd]; returns the values they are held as."""
        (kq, ks), (vq, vs) = quantize(k, self.gs), quantize(v, self.gs)
        self.k[pg, head, slot] = k_row_bytes(kq)
        units = self.v[pg, head].view(np.uint16).reshape(self.page // 4, 16, self.hd // 64, 4)
        for (m, u), x in v_row_units(vq).items():
            units[slot // 4, m, u, slot % 4] = x
        self.ks[pg, head, :, slot], self.vs[pg, head, :, slot] = ks, vs
        return values(kq, ks), values(vq, vs)

    def tensors(self, dev):
        return tuple(torch.from_numpy(x.copy()).to(dev) for x in (self.k, self.ks, self.v, self.vs))


def offsets(ns):
    return np.concatenate([[0], np.cumsum(ns)]).astype(np.int32)


def rope_tables(rows, hd, theta=1e4):
    a = np.arange(rows)[:, None] * theta ** (-np.arange(0, hd, 2) / hd)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def half(x):
    """binary64 -> binary16 as the library rounds everywhere: to binary32, then to binary16."""
    return x.astype(np.float32).astype(np.float16)


def same(got, want, label):
    """Bit equality, without printing the arrays."""
    got = got.cpu().numpy() if torch.is_tensor(got) else got
    assert got.shape == want.shape and got.dtype == want.dtype, f"{label}: {got.dtype}{got.shape} {want.dtype}{want.shape}"
    if got.dtype == np.float16:
        got, want = np.ascontiguousarray(got).view(np.uint16), np.ascontiguousarray(want).view(np.uint16)
    n = int(np.sum(got != want))
    assert n == 0, f"{label}: {n} of {got.size} differ"


def norm_rope(x, w, eps, cos, sin):
    """x fp16 [heads, hd] at one position: the row as binary64 before its last rounding."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
        x = half(x).astype(np.float64)
    lo, hi = np.split(x, 2, -1)
    c, s = cos.astype(np.float64), sin.astype(np.float64)
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)


def attention(q, k, v, last, scale):
    """q [n, NQ, hd], k, v [m, NKV, hd] (torch float64), query i sees keys 0 .. last[i]. Returns (out, bound): the exact
    result and the error a kernel may have, by the rules above."""
    n, NQ, hd = q.shape
    m, NKV = k.shape[0], k.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    if not m or not n:
        return out, bound + TINY
    key = torch.arange(m, device=q.device)
    seen = key[None] <= last[:, None]
    for h in range(NQ):
        kh, vh = k[:, h * NKV // NQ], v[:, h * NKV // NQ]
        z = torch.where(seen, q[:, h] @ kh.T * scale, -torch.inf)
        d = torch.where(seen, q[:, h].abs() @ kh.abs().T, 0).amax(-1, keepdim=True) * scale * (hd + 8) * E + 2.0 ** -21
        top = z.amax(-1, keepdim=True)
        p = torch.exp(z - torch.where(torch.isfinite(top), top, 0))
        tot = p.sum(-1, keepdim=True)
        tot = torch.where(tot > 0, tot, 1)
        o = p @ vh / tot
        A = p @ vh.abs() / tot
        far = seen.sum(-1, keepdim=True).double()
        out[:, h] = o
        bound[:, h] = U * o.abs() + (U + 2 * d + 2 * far * E) * A + TINY * (1 + far * vh.abs().amax() / tot)
    return out, bound


def assert_within(got, ref, bound, label):
    got = got.double()
    assert torch.isfinite(got).all(), f"{label}: not finite"
    over = ((got - ref).abs() - bound).max().item() if got.numel() else 0.0
    assert over <= 0, f"{label}: {over:.3e} over the bound, worst error {(got - ref).abs().max().item():.3e}"
