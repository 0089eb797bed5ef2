"""The oracle of the operators over microscaled blocks: numpy, 64 bits.

Element codes are kept one to a byte here (sign in the top bit of the type);
pack / tile functions restate the byte layouts of include/bz_mx.h and
include/bz_gemv.h.
"""

from __future__ import annotations

import numpy as np

BLOCK = 32
E2M1, E4M3 = "e2m1", "e4m3"
EMAX = {E2M1: 2, E4M3: 8}
SIGN = {E2M1: 8, E4M3: 128}


def grid(elem: str) -> np.ndarray:
    """Non-negative values of the type; a value's place is its code."""
    if elem == E2M1:
        return np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    codes = np.arange(127)
    e, m = codes >> 3, codes & 7
    return np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))


def quantize(x: np.ndarray, elem: str):
    """x float64 [M, K] -> (element codes uint8 [M, K], scale codes uint8 [M, K/32])."""
    g = grid(elem)
    M, K = x.shape
    v = x.reshape(M, K // BLOCK, BLOCK)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    amax = np.abs(v).max(-1)
    e = np.where(amax > 0, np.frexp(amax)[1] - 1 - EMAX[elem], -126)
    e = np.maximum(e, -126)
    y = np.ldexp(v, -e[..., None])
    mag = np.minimum(np.abs(y), g[-1])
    hi = np.clip(np.searchsorted(g, mag), 0, g.size - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = mag - g[lo], g[hi] - mag
    q = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    q = q + SIGN[elem] * np.signbit(y)
    return q.reshape(M, K).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray, elem: str) -> np.ndarray:
    """float64 [M, K] from element codes and scale codes."""
    g = grid(elem)
    mag = codes & (SIGN[elem] - 1)
    v = g[np.minimum(mag, g.size - 1)] * np.where(codes & SIGN[elem], -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * np.repeat(s, BLOCK, -1)


def rounded(x: np.ndarray, elem: str) -> np.ndarray:
    return values(*quantize(x, elem), elem)


def pack_nibbles(codes: np.ndarray) -> np.ndarray:
    """[M, K] -> [M, K/2], the even column in the low half."""
    return (codes[:, ::2] | codes[:, 1::2] << 4).astype(np.uint8)


def tile(codes: np.ndarray, scales: np.ndarray, elem: str, paired: bool = False) -> np.ndarray:
    """Element and scale codes [N, K], K % 128 == 0 -> tiled bytes.  Rows are
    rounded up to 16 with zeros; paired: gate rows 8b.. then up rows 8b.. a block."""
    N, K = codes.shape
    pad = -N % 16
    codes = np.pad(codes, ((0, pad), (0, 0)))
    zero = quantize(np.zeros((1, BLOCK)), elem)[1][0, 0]
    scales = np.pad(scales, ((0, pad), (0, 0)), constant_values=zero)
    rows, NU = codes.shape[0], K // 128
    out = []
    for b in range(rows // 16):
        r = np.arange(16) + 16 * b
        if paired:
            r = np.concatenate([np.arange(8) + 8 * b, np.arange(8) + 8 * b + N // 2])
        c = codes[r].reshape(16, NU, 128)
        if elem == E2M1:
            # piece g of row r at byte 256 g + 16 r of a tile
            t = pack_nibbles(c.reshape(16 * NU, 128)).reshape(16, NU, 4, 16).transpose(1, 2, 0, 3)
        else:
            # 16-k piece p at byte 1024 (p / 4) + 256 (p % 4) + 16 r
            t = c.reshape(16, NU, 8, 16).transpose(1, 2, 0, 3)
        s = np.zeros((-(-NU // 4) * 4, 4, 16), np.uint8)
        s[:NU] = scales[r].reshape(16, NU, 4).transpose(1, 2, 0)
        s = s.reshape(-1, 4, 64).transpose(0, 2, 1)  # four units a dword
        out.append(np.concatenate([t.reshape(-1), s.reshape(-1)]))
    return np.concatenate(out)


def rmsnorm_scale(x: np.ndarray, eps: float) -> np.ndarray:
    return 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def silu(g: np.ndarray) -> np.ndarray:
    return g / (1.0 + np.exp(-g))
