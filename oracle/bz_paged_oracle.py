"""CPU oracle of the operators over a paged key/value cache, in 64 bits, one row
after the other.  Test infrastructure only.

Arrays: pools [pages, HKV, page_size, D] as the values they stand for (codes
times scales), tables and lengths as integers.  Positions of a page outside
[0, pages) are not there.
"""

from __future__ import annotations

import numpy as np


def rows_of(T, B, kv_lens, q_starts):
    """(row, sequence, position) of every row that belongs to a sequence."""
    out = []
    for b in range(B):
        if q_starts is None:
            first, end = b, b + 1
        else:
            first = min(max(int(q_starts[b]), 0), T)
            end = min(max(int(q_starts[b + 1]), first), T)
        for t in range(first, end):
            out.append((t, b, max(int(kv_lens[b]), 0) - (end - t)))
    return out


def slot(table, j, ps, pages):
    """(page, place) of position j in a row of a page table, or None."""
    if j < 0 or j // ps >= len(table) or not 0 <= int(table[j // ps]) < pages:
        return None
    return int(table[j // ps]), j % ps


def norm_rope(x, w, eps, cos, sin):
    """x [..., D] -> rotated values and the magnitudes that rounding errors go with."""
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w
    h = x.shape[-1] // 2
    r = np.concatenate([-x[..., h:], x[..., :h]], -1)
    return x * cos + r * sin, np.abs(x * cos) + np.abs(r * sin)


def rope_cache(qkv, HQ, k_pages, v_pages, table, kv_lens, q_starts, cos, sin, positions=None, qn=None, kn=None,
               eps=1e-6):
    """q [T, HQ, D] (NaN in rows of no sequence) with magnitudes, and the pools' new
    values as {(page, place): (k, k magnitude, v)}, [HKV, D] each, before any
    rounding."""
    pages, HKV, ps, D = k_pages.shape
    T = qkv.shape[0]
    x = np.asarray(qkv, np.float64).reshape(T, HQ + 2 * HKV, D)
    q, mag, put = np.full((T, HQ, D), np.nan), np.zeros((T, HQ, D)), {}
    for t, b, pos in rows_of(T, len(kv_lens), kv_lens, q_starts):
        at = pos if positions is None else int(positions[t])
        if not 0 <= at < cos.shape[0]:
            q[t] = 0.0
            continue
        c, s = np.asarray(cos[at], np.float64), np.asarray(sin[at], np.float64)
        q[t], mag[t] = norm_rope(x[t, :HQ], qn, eps, c, s)
        where = slot(table[b], pos, ps, pages)
        if where is not None:
            put[where] = (*norm_rope(x[t, HQ:HQ + HKV], kn, eps, c, s), x[t, HQ + HKV:])
    return q, mag, put


def attention(q, k_pages, v_pages, table, kv_lens, q_starts=None, scale=None, prefix=None):
    """out [T, HQ, D] (NaN in rows of no sequence), sum_j w_j |v_j| of every output, and
    the largest sum_d |q_d k_d| scale of every head's row.  prefix: (table
    [groups, W], lens, seqs or None)."""
    pages, HKV, ps, D = k_pages.shape
    T, HQ, _ = q.shape
    G = HQ // HKV
    scale = D ** -0.5 if scale is None else scale
    q = np.asarray(q, np.float64)
    out, weight, size = np.full((T, HQ, D), np.nan), np.zeros((T, HQ, D)), np.zeros((T, HQ))
    for t, b, pos in rows_of(T, len(kv_lens), kv_lens, q_starts):
        keys = []
        if prefix is not None:
            ptable, plens, pseqs = prefix
            for g in range(len(plens)):
                if pseqs is None or pseqs[g] <= b < pseqs[g + 1]:
                    keys += [slot(ptable[g], j, ps, pages) for j in range(int(plens[g]))]
                    break
        keys += [slot(table[b], j, ps, pages) for j in range(pos + 1)]
        keys = [k for k in keys if k is not None]
        if not keys:
            out[t] = 0.0
            continue
        pg, at = np.array(keys).T
        for h in range(HQ):
            k = k_pages[pg, h // G, at].astype(np.float64)
            v = v_pages[pg, h // G, at].astype(np.float64)
            s = (k @ q[t, h]) * scale
            e = np.exp(s - s.max())
            w = e / e.sum()
            out[t, h] = w @ v
            weight[t, h] = w @ np.abs(v)
            size[t, h] = (np.abs(k) @ np.abs(q[t, h])).max() * scale
    return out, weight, size
