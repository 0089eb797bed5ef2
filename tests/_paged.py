"""Cases over a paged cache, their oracle and its tolerances (not collected)."""

from __future__ import annotations

import numpy as np
import torch

from oracle import bz_paged_oracle as P

E4M3 = torch.float8_e4m3fn
BF16 = torch.bfloat16


def starts_of(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


class Cache:
    """A pool full of random values; tables of pages in random order."""

    def __init__(self, rng, pages, HKV, ps, D, kv="bf16", layout="hnd", dev="cuda"):
        self.pages, self.HKV, self.ps, self.D, self.kv, self.dev, self.rng = pages, HKV, ps, D, kv, dev, rng
        self.free = list(rng.permutation(pages))
        pools = []
        for _ in range(2):
            a = torch.from_numpy(rng.standard_normal((pages, HKV, ps, D)).astype(np.float32)).to(dev)
            scale = None
            if kv == "e4m3":
                scale = torch.from_numpy(rng.uniform(0.005, 0.02, HKV).astype(np.float32)).to(dev)
                a = (a / scale[:, None, None]).clamp(-448, 448).to(E4M3)
            else:
                a = a.to(BF16)
            if layout == "nhd":  # [pages, ps, HKV, D] behind a transposed view
                a = a.transpose(1, 2).contiguous().transpose(1, 2)
            elif layout == "pair":  # keys and values of a page side by side
                a = torch.stack([a.view(torch.uint8) if kv == "e4m3" else a] * 2, 1)
                a = a.view(E4M3)[:, 1] if kv == "e4m3" else a[:, 1]
            pools.append((a, scale))
        (self.k, self.k_scale), (self.v, self.v_scale) = pools

    def table(self, rows, width, pad=0):
        """[rows, width] distinct pages, of a tensor that is `pad` entries wider."""
        ids = np.array([self.free.pop() for _ in range(rows * width)], np.int32).reshape(rows, width)
        t = torch.from_numpy(np.concatenate([ids, np.full((rows, pad), -7, np.int32)], 1)).to(self.dev)
        return t[:, :width]

    def values(self, which):
        pool, scale = (self.k, self.k_scale) if which == "k" else (self.v, self.v_scale)
        a = pool.to(torch.float32).cpu().double()
        return (a if scale is None else a * scale.cpu().double()[:, None, None]).numpy()

    def raw(self, which):
        pool = self.k if which == "k" else self.v
        return (pool.view(torch.uint8) if self.kv == "e4m3" else pool.view(torch.int16)).cpu().numpy()


def ints(a, dev="cuda"):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


def bf16(a, dev="cuda"):
    return torch.from_numpy(np.asarray(a, np.float32)).to(BF16).to(dev)


def attention_bound(out, weight, size, D):
    """How far a bf16 output may be from the 64-bit one.

    out is rounded once (half a bf16 step, 2^-8 of it); a probability may be rounded
    to bf16 before its product with the value (2^-8 of w |v|); a score is a sum of
    D products in fp32 (error D 2^-24 sum |q k| scale, scaled and its maximum
    subtracted with two more roundings of 2^-24 of the same), which changes each
    weight, and their sum, by that share; exponentials, sums and the merge of parts
    are in fp32: 2^-16 covers some hundred of their roundings."""
    score = (D + 4) * 2.0 ** -24 * size[..., None]
    return 2.0 ** -8 * np.abs(out) + (2.0 ** -8 + 2 * score + 2.0 ** -16) * weight + 1e-30


def check_attention(got, q, cache, table, kv_lens, q_starts=None, scale=None, prefix=None, before=None):
    """got [T, HQ D] against the oracle; rows of no sequence equal `before`."""
    ref, weight, size = P.attention(q.float().cpu().numpy(), cache.values("k"), cache.values("v"),
                                    table.cpu().numpy(), kv_lens, q_starts, scale, prefix)
    g = got.float().cpu().double().numpy().reshape(ref.shape)
    none = np.isnan(ref[:, 0, 0])
    if before is not None:
        np.testing.assert_array_equal(got.view(torch.int16).cpu().numpy()[none],
                                      before.view(torch.int16).cpu().numpy()[none])
    ref, g, weight, size = ref[~none], g[~none], weight[~none], size[~none]
    bound = attention_bound(ref, weight, size, cache.D)
    off = np.abs(g - ref) - bound
    assert np.isfinite(g).all() and (off <= 0).all(), \
        f"off by {np.abs(g - ref).max():.3g}, at most {bound.flat[off.argmax()]:.3g} there: {np.argwhere(off > 0)[:4]}"
