"""How near few rows' attention over a paged cache comes to the 64-bit one, whose probabilities go into their
products as two bf16 parts (not collected).

The first part is a probability cut to 8 bits, the second the rest (below 2^-7 of it) rounded to 8
bits, at most 2^-8 of the rest: 2^-15 of the probability is lost.  A score is a sum of D products in fp32
(D 2^-24 sum |q k| scale, and two more roundings), which changes each weight, and their sum, by that share.
The sums over n keys may be cut in the matrix cores, 2^-23 of them each, in numerator and denominator.
Exponentials, rescaling and the merge of parts: 2^-16 covers some hundred fp32 roundings.  Then one
rounding to bf16, of half a step where the value lies."""

from __future__ import annotations

import numpy as np

from oracle import bz_paged_oracle as P


def half_step(x):
    """Half a bf16 step at |x|."""
    _, e = np.frexp(np.maximum(np.abs(x), 1e-37))  # |x| in [2^(e-1), 2^e)
    return np.ldexp(1.0, e - 9)


def parts_bound(out, weight, size, D, keys):
    e = (2.0 ** -15 + 2 * (D + 4) * 2.0 ** -24 * size[..., None] + keys * 2.0 ** -22 + 2.0 ** -16) * weight
    return half_step(np.abs(out) + e) + e


def check_parts(got, q, cache, table, kv_lens, q_starts=None, scale=None, prefix=None):
    """got [T, HQ D] against the oracle."""
    ref, weight, size = P.attention(q.float().cpu().numpy(), cache.values("k"), cache.values("v"),
                                    table.cpu().numpy(), kv_lens, q_starts, scale, prefix)
    g = got.float().cpu().double().numpy().reshape(ref.shape)
    keys = max(kv_lens) + (0 if prefix is None else max(prefix[1]))
    off = np.abs(g - ref) - parts_bound(ref, weight, size, cache.D, keys)
    assert np.isfinite(g).all() and (off <= 0).all(), f"off by up to {off.max():.3g} more than it may: {np.argwhere(off > 0)[:4]}"


KEYS, PROB, VALUE = 101, 0.501953125, 1.75


def midway(cache, table):
    """Keys of one sequence of KEYS positions, and the scale, with which a query of ones in column 0 has a probability
    of 1 at the first and PROB, midway between two bf16 numbers, at the others (before the division by
    their sum), values of VALUE: one bf16 part of PROB, cut or rounded, changes the output by a step."""
    cache.k.zero_()
    cache.k[int(table[0, 0]), :, 0, 0] = 1.0
    cache.v.fill_(VALUE)
    return -float(np.log(PROB))
