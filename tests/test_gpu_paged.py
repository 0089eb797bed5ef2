"""The operators over a paged cache on the GPU, against the 64-bit oracle.

Tolerances: tests/_paged.py for attention.  A rotated value is rounded once (half
a step: bf16 2^-8, e4m3 2^-4 of it, or half of e4m3's smallest step 2^-9 times the
scale); its fp32 steps (a sum of D squares, root, quotient, four products, a
sum: at most D / 2 + 8 roundings of 2^-24, as the squares' errors halve) are far
below 2^-16 of its terms' magnitude."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from oracle import bz_paged_oracle as P
from tests._paged import BF16, Cache, bf16, check_attention, ints, starts_of
from tests._paged_parts import KEYS, check_parts, midway

from breeze_amd import paged as T

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _tables(rng, rows, D, dtype):
    th = rng.uniform(-4, 4, (rows, D // 2)).astype(np.float32)
    # halves that differ, as an operator may not assume that they are alike
    cos = torch.from_numpy(np.concatenate([np.cos(th), np.cos(th + 0.1)], -1)).to(dtype).to(DEV)
    sin = torch.from_numpy(np.concatenate([np.sin(th), np.sin(th + 0.1)], -1)).to(dtype).to(DEV)
    return cos, sin


def _append(rng, cache, HQ, table, kv_lens, n, *, norms=True, cs=torch.float32, positions=None, rows=None, before=0,
            behind=0, cs_rows=None):
    """One call and its check; returns what it was given."""
    q_starts = None if n is None else starts_of(n) + before
    T_ = len(kv_lens) if n is None else int(q_starts[-1]) + behind
    D, HKV = cache.D, cache.HKV
    qkv = bf16(rng.standard_normal((T_, (HQ + 2 * HKV) * D)) * 2)
    cos, sin = _tables(rng, cs_rows or max(max(kv_lens), 1), D, cs)
    qn, kn = (bf16(1 + 0.1 * rng.standard_normal(D)) for _ in range(2)) if norms else (None, None)
    old = {w: cache.raw(w).copy() for w in "kv"}
    q_out = bf16(rng.standard_normal((T_, HQ, D)))
    q_before = q_out.clone()
    got = T.paged_rope_cache(qkv, cos, sin, cache.k, cache.v, table, ints(kv_lens), HQ,
                             None if n is None else ints(q_starts), q_norm_w=qn, k_norm_w=kn, eps=1e-6,
                             positions=None if positions is None else torch.tensor(positions, device=DEV),
                             k_scale=cache.k_scale, v_scale=cache.v_scale, q_out=q_out)
    assert got is q_out
    f = lambda t: None if t is None else t.float().cpu().double().numpy()  # noqa: E731
    ref, mag, put = P.rope_cache(f(qkv), HQ, cache.values("k"), cache.values("v"), table.cpu().numpy(), kv_lens,
                                 q_starts, f(cos), f(sin), positions, f(qn), f(kn), 1e-6)
    g = f(got)
    none = np.isnan(ref[:, 0, 0])
    np.testing.assert_array_equal(g[none], f(q_before)[none])
    assert (np.abs(g - ref)[~none] <= (2.0 ** -8 * np.abs(ref) + 2.0 ** -16 * mag)[~none] + 1e-30).all()
    for w, scale in (("k", cache.k_scale), ("v", cache.v_scale)):
        new, touched = cache.raw(w), np.zeros((cache.pages, cache.ps), bool)
        vals = cache.values(w)
        for (page, at), (k, k_mag, v) in put.items():
            touched[page, at] = True
            want, m = (k, k_mag) if w == "k" else (v, np.abs(v))
            if scale is None:
                tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -16 * m
                if w == "v":
                    tol = np.zeros_like(want)  # a copy
            else:
                sc = f(scale)[:, None]
                want = np.clip(want, -448 * sc, 448 * sc)
                tol = np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * sc) + 2.0 ** -16 * m
            assert (np.abs(vals[page, :, at] - want) <= tol + 1e-30).all(), (w, page, at)
        keep = ~np.broadcast_to(touched[:, None, :, None], new.shape)
        np.testing.assert_array_equal(new[keep], old[w][keep])
    return qkv, got


HEADS = [(16, 8, 128), (8, 2, 128), (16, 4, 256), (6, 2, 64), (5, 5, 64), (16, 1, 128), (9, 3, 256), (1, 1, 128)]


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", HEADS)
def test_append_steps(HQ, HKV, D, kv):
    rng = np.random.default_rng(HQ * 1000 + D)
    cache = Cache(rng, 20, HKV, 16, D, kv)
    table = cache.table(3, 5, pad=2)
    _append(rng, cache, HQ, table, [1, 17, 80], None)


@pytest.mark.parametrize("cs", [torch.float32, BF16])
@pytest.mark.parametrize("norms", [True, False])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "pair"])
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_append_prompts(kv, layout, norms, cs):
    """Ragged new rows, an empty sequence among them, rows of no sequence on both ends,
    rows at negative positions."""
    rng = np.random.default_rng(5)
    cache = Cache(rng, 40, 2, 32, 128, kv, layout)
    table = cache.table(5, 4)
    _append(rng, cache, 6, table, [37, 9, 5, 128, 64], [37, 3, 0, 100, 70], norms=norms, cs=cs, before=2, behind=3)


def test_append_many_sequences():
    """More sequences than a wave has lanes."""
    rng = np.random.default_rng(6)
    cache = Cache(rng, 310, 1, 16, 64)
    table = cache.table(150, 2)
    n = rng.integers(0, 4, 150)
    _append(rng, cache, 2, table, list(rng.integers(3, 33, 150)), n, behind=1)


def test_append_positions():
    """Rotary rows apart from the places; rows outside the rotary table and pages that
    are not there write nothing."""
    rng = np.random.default_rng(7)
    cache = Cache(rng, 20, 2, 16, 64)
    table = cache.table(4, 3)
    table[1, 0] = -1
    table[2, 2] = 20
    table[3, 1] = 2 ** 31 - 1
    _append(rng, cache, 4, table, [5, 16, 48, 60], [2, 4, 20, 20], cs_rows=50,
            positions=list(range(40, 46)) + list(range(-3, 17)) + list(range(35, 55)))


def test_append_saturates_and_keeps_nan():
    cache = Cache(np.random.default_rng(8), 2, 1, 16, 64, "e4m3")
    cache.k_scale.fill_(1.0)
    cache.v_scale.fill_(0.5)
    x = torch.zeros(1, 3 * 64, device=DEV, dtype=BF16)
    x[0, 64:70] = torch.tensor([500.0, -1e30, float("inf"), float("nan"), 447.0, -0.0009])
    x[0, 128:133] = torch.tensor([230.0, -float("inf"), float("nan"), 224.0, 0.0004])
    one, zero = torch.ones(1, 64, device=DEV), torch.zeros(1, 64, device=DEV)
    T.paged_rope_cache(x, one, zero, cache.k, cache.v, ints([[1]]), ints([1]), 1, k_scale=cache.k_scale,
                       v_scale=cache.v_scale)
    k, v = cache.k.float()[1, 0, 0].tolist(), cache.v.float()[1, 0, 0].tolist()
    # (the partner columns are zero times a sine of zero; an infinity's would be NaN there, not here)
    assert k[:3] == [448.0, -448.0, 448.0] and k[3] != k[3] and k[4] == 448.0 and k[5] == -0.0
    assert v[0] == 448.0 and v[1] == -448.0 and v[2] != v[2] and v[3] == 448.0 and v[4] == 0.0


def _attend(seed, HQ, HKV, D, kv_lens, n=None, ps=16, kv="bf16", layout="hnd", prefix=None, spread=1.5, width=None,
            before=0, behind=0, edit=None, scale=None):
    rng = np.random.default_rng(seed)
    B = len(kv_lens)
    width = width or max(1, -(-max(kv_lens) // ps))
    pw = 0 if prefix is None else max(1, -(-max(prefix[0]) // ps))
    cache = Cache(rng, B * width + (0 if prefix is None else len(prefix[0]) * pw) + 1, HKV, ps, D, kv, layout)
    table = cache.table(B, width, pad=1)
    q_starts = None if n is None else starts_of(n) + before
    rows = B if n is None else int(q_starts[-1]) + behind
    q = bf16(rng.standard_normal((rows, HQ, D)) * spread)
    out = bf16(rng.standard_normal((rows, HQ * D)))
    old = out.clone()
    args = {"scale": scale, "k_scale": cache.k_scale, "v_scale": cache.v_scale, "out": out}
    starts = None if n is None else ints(q_starts)
    ref_prefix = None
    if prefix is not None:
        lens, seqs = prefix
        ptable = cache.table(len(lens), pw, pad=3)
        ref_prefix = (ptable.cpu().numpy(), lens, seqs)
    if edit is not None:
        edit(cache, table)
        if prefix is not None:
            ref_prefix = (ptable.cpu().numpy(), lens, seqs)
    if prefix is None:
        got = T.paged_attention(q, cache.k, cache.v, table, ints(kv_lens), starts, **args)
    else:
        got = T.shared_prefix_attention(q, cache.k, cache.v, ptable, ints(lens), table, ints(kv_lens), starts,
                                        None if seqs is None else ints(seqs), **args)
    assert got is out
    check_attention(got, q, cache, table, kv_lens, q_starts, scale, ref_prefix, old)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", HEADS)
def test_attend_steps(HQ, HKV, D, kv):
    _attend(HQ + D, HQ, HKV, D, [1, 2, 15, 16, 17, 33, 130, 0], kv=kv)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", [(16, 8, 128), (16, 4, 256), (7, 1, 64)])
def test_attend_long_steps(HQ, HKV, D, kv):
    """Contexts that are split, next to short and empty ones."""
    _attend(1, HQ, HKV, D, [3001, 5, 0, 1024, 257], ps=64, kv=kv)


@pytest.mark.parametrize("ps", [16, 32, 128, 4096])
def test_attend_page_sizes(ps):
    _attend(2, 4, 2, 128, [200, 31, 129], ps=ps)


@pytest.mark.parametrize("layout", ["nhd", "pair"])
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_attend_layouts(kv, layout):
    _attend(3, 6, 3, 128, [70, 300], n=[3, 40], ps=32, kv=kv, layout=layout)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", HEADS)
def test_attend_several_rows(HQ, HKV, D, kv):
    """Drafted tokens: every row sees one position more; rows before the sequence's
    first position (n above the length), no rows, and rows of no sequence."""
    _attend(4, HQ, HKV, D, [40, 3, 9, 100, 0], n=[5, 5, 0, 7, 2], kv=kv, before=1, behind=2)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", [(4, 2, 128), (4, 1, 256), (3, 1, 64), (2, 2, 128), (16, 1, 64)])
def test_attend_prompts(HQ, HKV, D, kv):
    """Prompts and chunks of them: lengths around the tiles' sizes."""
    _attend(5, HQ, HKV, D, [131, 64, 257, 200, 1], n=[131, 64, 63, 129, 1], kv=kv)


def test_attend_a_longer_prompt():
    _attend(6, 4, 2, 128, [700, 513], n=[700, 33], ps=64)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", [(16, 1, 64), (4, 2, 128), (6, 2, 128), (8, 1, 256)])
def test_attend_prompts_of_several_parts(HQ, HKV, D, kv):
    """Chunks of prompts whose tiles' keys are cut, so that the last workgroup of a tile joins them; a sequence
    with nothing before it, one row, fewer positions than rows, and none among them."""
    _attend(26, HQ, HKV, D, [1500, 333, 1, 40, 0, 901], n=[200, 333, 1, 50, 3, 70], kv=kv, ps=32, before=1, behind=1)


@pytest.mark.parametrize("HQ,HKV,D,n", [(8, 8, 64, [1] * 2200), (144, 9, 64, [3] * 1100)])
def test_attend_more_tiles_than_counters(HQ, HKV, D, n):
    """So many tiles that a launch of its own joins their parts.  The sequences share pages."""
    rng = np.random.default_rng(27)
    B, ps = len(n), 64
    cache = Cache(rng, 48, HKV, ps, D)
    table = ints(rng.integers(0, 48, (B, 6)))
    lens = rng.integers(0, 20, B)
    lens[::100] = rng.integers(300, 385, len(lens[::100]))
    q = bf16(rng.standard_normal((sum(n), HQ, D)))
    starts = starts_of(n)
    got = T.paged_attention(q, cache.k, cache.v, table, ints(lens), ints(starts))
    check_attention(got, q, cache, table, lens, starts)


def test_attend_many_sequences():
    rng = np.random.default_rng(9)
    _attend(7, 2, 1, 64, list(rng.integers(0, 40, 150)), n=rng.integers(0, 4, 150), behind=1)


def test_attend_a_table_that_is_too_short():
    """Positions behind the table's pages are not there."""
    _attend(8, 4, 2, 64, [70, 100, 33], n=[3, 40, 1], width=3, ps=16)


def test_attend_pages_that_are_not_there():
    def edit(cache, table):
        table[0, 1] = -1
        table[1, 0] = cache.pages
        table[2, :] = -5
        table[3, 3] = 2 ** 31 - 1

    _attend(9, 4, 2, 128, [60, 16, 40, 130], n=[1, 1, 9, 100], edit=edit, width=9)
    _attend(9, 4, 2, 128, [60, 16, 40, 130], edit=edit, width=9)


@pytest.mark.parametrize("HQ,HKV,D,kv", [(4, 2, 64, "e4m3"), (16, 2, 128, "e4m3"), (8, 1, 256, "e4m3"), (8, 1, 256, "bf16")])
def test_attend_chunks_with_pages_that_are_not_there(HQ, HKV, D, kv):
    """In the middle of a tile of keys, a whole tile, the first and the last."""
    def edit(cache, table):
        table[0, 1:7] = -1
        table[0, 30] = cache.pages
        table[1, 0] = -2
        table[1, 36] = 2 ** 31 - 1
        table[2, :] = -5

    _attend(30, HQ, HKV, D, [700, 599, 300], n=[140, 20, 40], kv=kv, edit=edit, width=44)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("layout", ["nhd", "pair"])
def test_attend_chunks_of_other_layouts(kv, layout):
    _attend(31, 8, 2, 128, [500, 260], n=[100, 260], kv=kv, layout=layout)
    _attend(32, 8, 2, 64, [500, 260], n=[100, 20], kv=kv, layout=layout, ps=64)


@pytest.mark.parametrize("spread,scale", [(12.0, None), (0.0, None), (1.0, 30.0), (3.0, 1e-4)])
def test_attend_scales(spread, scale):
    """One key that takes all, keys that weigh alike, and other scales."""
    _attend(10, 4, 2, 128, [300, 70], n=[2, 70], spread=spread, scale=scale)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", [(16, 8, 128), (16, 4, 256), (6, 2, 64), (16, 1, 128)])
def test_prefix_steps(HQ, HKV, D, kv):
    """Two prefixes; a sequence of none; own lengths of zero."""
    _attend(11, HQ, HKV, D, [1, 0, 40, 17, 5], kv=kv, prefix=([100, 33], [0, 3, 4]))


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_prefix_of_all(kv):
    rng = np.random.default_rng(12)
    _attend(12, 16, 8, 128, list(rng.integers(0, 90, 40)), kv=kv, ps=32, prefix=([1000], None))


@pytest.mark.parametrize("lens", [[0], [1], [16], [15], [257]])
def test_prefix_lengths(lens):
    _attend(13, 8, 2, 128, [3, 0, 20], prefix=(lens, None))


def test_prefix_several_rows():
    """Drafted tokens and prompts behind prefixes, empty groups and sequences among them."""
    _attend(14, 6, 2, 64, [5, 90, 0, 1, 30], n=[5, 80, 0, 2, 1], prefix=([70, 10, 300], [0, 2, 2, 5]), before=1,
            behind=2)


def test_prefix_many_sequences():
    rng = np.random.default_rng(15)
    _attend(15, 2, 1, 64, list(rng.integers(0, 20, 130)), n=rng.integers(0, 3, 130),
            prefix=([200, 60], [0, 70, 128]))


@pytest.mark.parametrize("HQ,HKV,D", [(16, 8, 128), (16, 1, 64), (4, 4, 128), (9, 3, 128), (16, 4, 256)])
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_prefix_many_groups(HQ, HKV, D, kv):
    """One row each: prefixes of one sequence to 33, and of none, sequences before, between and behind them; more
    segments than one wave counts at a time."""
    rng = np.random.default_rng(16)
    size = [1, 2, 0, 33, 1, 5, 8, 0, 3, 4, 9, 1, 1, 2]
    starts = 2 + np.cumsum([0] + size)
    B = int(starts[-1]) + 3
    for _ in range(2):  # (the second time with the counters that the first has left)
        _attend(17, HQ, HKV, D, list(rng.integers(0, 400, B)), kv=kv, prefix=(list(rng.integers(0, 700, len(size))),
                                                                           [int(s) for s in starts]))


def test_starts_that_decrease_leave_the_workspace_usable():
    """What such rows hold is not said; the next call with good ones is right."""
    rng = np.random.default_rng(18)
    cache = Cache(rng, 64, 2, 16, 128)
    table, ptable = cache.table(8, 4), cache.table(3, 4)
    q = bf16(rng.standard_normal((8, 4, 128)))
    lens = ints([50, 9, 64, 1, 0, 33, 20, 64])
    good = (lambda: T.shared_prefix_attention(q, cache.k, cache.v, ptable, ints([60, 64, 7]), table, lens,
                                              prefix_seqs=ints([0, 3, 3, 7])),
            lambda: T.paged_attention(q, cache.k, cache.v, table, lens, ints([0, 2, 3, 3, 5, 6, 7, 8, 8])))
    want = [f() for f in good]
    T.shared_prefix_attention(q, cache.k, cache.v, ptable, ints([60, 64, 7]), table, lens, prefix_seqs=ints([0, 8, 0, 8]))
    T.paged_attention(q, cache.k, cache.v, table, lens, ints([0, 8, 0, 8, 0, 8, 0, 8, 2]))
    for f, w in zip(good, want):
        assert torch.equal(f(), w)


def _poison(cache, table, kv_lens):
    """NaN and infinities in every place of the pool that no position of these
    sequences has."""
    used = np.zeros((cache.pages, cache.ps), bool)
    for b, n in enumerate(kv_lens):
        for j in range(n):
            used[int(table[b, j // cache.ps]), j % cache.ps] = True
    where = torch.from_numpy(~used).to(cache.k.device)[:, None, :, None]
    for pool in (cache.k, cache.v):
        if cache.kv == "e4m3":
            pool.view(torch.uint8).copy_(torch.where(where, torch.tensor(0x7F, dtype=torch.uint8, device=DEV),
                                                     pool.view(torch.uint8)))
        else:
            bad = torch.where(torch.arange(cache.D, device=DEV) % 2 == 0, float("nan"), float("-inf")).to(BF16)
            pool.copy_(torch.where(where, bad, pool))


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", [(4, 2, 128), (8, 2, 64), (4, 1, 256)])
@pytest.mark.parametrize("n", [None, [1, 9, 20, 130]])
def test_places_behind_the_length_have_no_part(HQ, HKV, D, kv, n):
    lens = [5, 16, 75, 300]
    _attend(16, HQ, HKV, D, lens, n=n, kv=kv, ps=32, edit=lambda c, t: _poison(c, t, lens))


@pytest.mark.parametrize("rows", [5, 150])
@pytest.mark.parametrize("bad", ["k", "v", "both"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_later_rows_have_no_part(value, bad, rows):
    """The last token's key or value is not finite: the rows before it are as if it were
    not there, bit for bit its own run without it would allow."""
    HQ, HKV, D, ps, lens = 4, 2, 128, 16, [rows + 30]
    rng = np.random.default_rng(17)
    cache = Cache(rng, 20, HKV, ps, D)
    table = cache.table(1, 12)
    q = bf16(rng.standard_normal((rows, HQ, D)))
    j = lens[0] - 1
    if bad != "v":
        cache.k[int(table[0, j // ps]), :, j % ps, 3] = value
    if bad != "k":
        cache.v[int(table[0, j // ps]), :, j % ps, ::5] = value
    out = T.paged_attention(q, cache.k, cache.v, table, ints(lens), ints([0, rows]))
    ref, weight, size = P.attention(q[:-1].float().cpu().numpy(), cache.values("k"), cache.values("v"),
                                    table.cpu().numpy(), [j], [0, rows - 1])
    from tests._paged import attention_bound

    got = out[:-1].float().cpu().double().numpy().reshape(ref.shape)
    assert (np.abs(got - ref) <= attention_bound(ref, weight, size, D)).all()
    last = out[-1].float().cpu().numpy().reshape(HQ, D)
    if bad == "v":  # the row itself attends it: its columns are what it is, the others finite
        hit = np.isnan(last) if np.isnan(value) else last == value
        assert hit[:, ::5].all() and np.isfinite(np.delete(last, np.s_[::5], 1)).all()
    elif np.isnan(value):
        assert np.isnan(last).all()


@pytest.mark.parametrize("HQ,HKV,D,kv", [(4, 2, 128, "bf16"), (16, 1, 64, "e4m3"), (8, 1, 256, "bf16"), (8, 1, 256, "e4m3")])
def test_later_rows_have_no_part_in_parts(HQ, HKV, D, kv):
    """The same where a tile's keys are cut, the bad token in the last chunk, and further rows behind it."""
    rows, ps = 150, 32
    rng = np.random.default_rng(29)
    cache = Cache(rng, 60, HKV, ps, D, kv)
    table = cache.table(1, 40)
    q = bf16(rng.standard_normal((rows, HQ, D)))
    length, j = 1200, 1150  # position j is row 100
    bits = cache.v.view(torch.uint8) if kv == "e4m3" else cache.v.view(torch.int16)
    bits[int(table[0, j // ps]), :, j % ps, ::3] = 0x7F if kv == "e4m3" else 0x7FC0
    scales = {"k_scale": cache.k_scale, "v_scale": cache.v_scale}
    out = T.paged_attention(q, cache.k, cache.v, table, ints([length]), ints([0, rows]), **scales)
    ref, weight, size = P.attention(q[:100].float().cpu().numpy(), cache.values("k"), cache.values("v"),
                                    table.cpu().numpy(), [j], [0, 100])
    from tests._paged import attention_bound

    got = out[:100].float().cpu().double().numpy().reshape(ref.shape)
    assert (np.abs(got - ref) <= attention_bound(ref, weight, size, D)).all()
    later = out[100:].float().cpu().numpy().reshape(50, HQ, D)
    assert np.isnan(later[:, :, ::3]).all() and np.isfinite(np.delete(later, np.s_[::3], 2)).all()


def test_keys_of_minus_infinity_scores():
    """A score of -inf weighs nothing next to a finite one; a row of nothing else has no
    softmax: NaN."""
    cache = Cache(np.random.default_rng(18), 4, 1, 16, 64)
    table = cache.table(1, 2)
    cache.k[:, :, :, 0] = -float("inf")
    cache.k[int(table[0, 1]), 0, 3, 0] = 0.0
    q = torch.ones(20, 1, 64, device=DEV, dtype=BF16)
    out = T.paged_attention(q, cache.k, cache.v, table, ints([20]), ints([0, 20])).float()
    assert torch.isnan(out[:19]).all()
    torch.testing.assert_close(out[19], cache.v[int(table[0, 1]), 0, 3].float(), rtol=2.0 ** -8, atol=0)


def test_offsets_beyond_32_bits():
    """Pages more than 4 GiB into the pool."""
    HQ, HKV, D, ps = 4, 2, 128, 256
    pages = (5 << 30) // (HKV * ps * D * 2)
    k, v = (torch.empty(pages, HKV, ps, D, device=DEV, dtype=BF16) for _ in range(2))
    table = ints([[pages - 1, 3, pages - 2]])
    g = torch.Generator(device=DEV).manual_seed(1)
    for p in table[0].tolist():
        for pool in (k, v):
            pool[p] = torch.randn(HKV, ps, D, device=DEV, generator=g).to(BF16)
    small = Cache(np.random.default_rng(19), 3, HKV, ps, D)
    small.k, small.v = (pool[table[0].long()].contiguous() for pool in (k, v))
    for n in (1, 40):
        q = torch.randn(n, HQ, D, device=DEV, generator=g).to(BF16)
        got = T.paged_attention(q, k, v, table, ints([700]), ints([0, n]))
        want = T.paged_attention(q, small.k, small.v, ints([[0, 1, 2]]), ints([700]), ints([0, n]))
        assert torch.equal(got, want)
        check_attention(got, q, small, ints([[0, 1, 2]]), [700], [0, n])
    cos, sin = _tables(np.random.default_rng(20), 768, D, torch.float32)
    qkv = torch.randn(1, (HQ + 2 * HKV) * D, device=DEV, generator=g).to(BF16)
    T.paged_rope_cache(qkv, cos, sin, k, v, table, ints([701]), HQ)
    T.paged_rope_cache(qkv, cos, sin, small.k, small.v, ints([[0, 1, 2]]), ints([701]), HQ)
    for pool, s in ((k, small.k), (v, small.v)):
        assert torch.equal(pool[table[0].long()], s)


def _session(seed, kv="bf16", HQ=8, HKV=2, D=128, ps=16, prefix=40):
    """Buffers of a small served batch: three sequences behind a shared prefix."""
    rng = np.random.default_rng(seed)
    cache = Cache(rng, 60, HKV, ps, D, kv)
    return rng, cache, cache.table(1, 4), cache.table(3, 8), prefix


def _whole(qkv, HQ, HKV, D, cos, sin, qn, kn):
    """Rotated q and k, and v, of a whole sequence in 64 bits."""
    x = qkv.float().cpu().double().numpy().reshape(-1, HQ + 2 * HKV, D)
    c, s = (t.float().cpu().double().numpy()[: len(x), None] for t in (cos, sin))
    w = [t.float().cpu().double().numpy() for t in (qn, kn)]
    return P.norm_rope(x[:, :HQ], w[0], 1e-6, c, s)[0], P.norm_rope(x[:, HQ:HQ + HKV], w[1], 1e-6, c, s)[0], x[:, HQ + HKV:]


def test_a_served_batch():
    """Prefix, prompts of different lengths, then steps and drafted tokens, all through
    the operators: every row's attention against the whole sequence's from the raw
    qkv.  The cache holds k rounded to bf16 (2^-8 of each), q likewise: a score is
    off by at most 2 * 2^-8 sum |q k| scale, which changes a weight by that share."""
    HQ, HKV, D = 8, 2, 128
    rng, cache, ptable, table, prefix = _session(21)
    cos, sin = _tables(rng, 200, D, torch.float32)
    qn, kn = (bf16(1 + 0.1 * rng.standard_normal(D)) for _ in range(2))
    width = (HQ + 2 * HKV) * D
    shared = bf16(rng.standard_normal((prefix, width)))
    raw = [[shared] for _ in range(3)]
    outs = [[] for _ in range(3)]
    norms = {"q_norm_w": qn, "k_norm_w": kn}
    q = T.paged_rope_cache(shared, cos, sin, cache.k, cache.v, ptable, ints([prefix]), HQ, ints([0, prefix]), **norms)
    first = T.paged_attention(q, cache.k, cache.v, ptable, ints([prefix]), ints([0, prefix]))
    lens = np.zeros(3, int)
    for n in ([33, 1, 70], [1, 1, 1], [1, 1, 1], [4, 2, 1], [1, 0, 5]):
        lens += n
        new = [bf16(rng.standard_normal((m, width))) for m in n]
        starts = starts_of(n)
        at = np.concatenate([np.arange(prefix + l - m, prefix + l) for l, m in zip(lens, n)])
        q = T.paged_rope_cache(torch.cat(new), cos, sin, cache.k, cache.v, table, ints(lens), HQ, ints(starts),
                               positions=torch.from_numpy(at).to(DEV), **norms)
        out = T.shared_prefix_attention(q, cache.k, cache.v, ptable, ints([prefix]), table, ints(lens), ints(starts))
        for b in range(3):
            raw[b].append(new[b])
            outs[b].append(out[starts[b]:starts[b + 1]])
    for b in range(3):
        qf, kf, vf = _whole(torch.cat(raw[b]), HQ, HKV, D, cos, sin, qn, kn)
        got = torch.cat([first] + outs[b]).float().cpu().double().numpy().reshape(-1, HQ, D)
        for t in range(len(got)):
            for h in range(HQ):
                k, v = kf[: t + 1, h // 4], vf[: t + 1, h // 4]
                s = k @ qf[t, h] * D ** -0.5
                w = np.exp(s - s.max())
                w /= w.sum()
                size = (np.abs(k) @ np.abs(qf[t, h])).max() * D ** -0.5
                ref, mag = w @ v, w @ np.abs(v)
                bound = 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2 * 2 * 2.0 ** -8 * size) * mag + 2.0 ** -16 * mag
                assert (np.abs(got[t, h] - ref) <= bound).all(), (b, t, h)


def test_replayed_steps_follow_the_lengths():
    """A captured step whose lengths and positions advance on the device: each replay is
    the eager step, with eager work between the replays.  Two graphs that interleave keep
    their results apart."""
    HQ, HKV, D = 8, 2, 128
    rng, cache, ptable, table, prefix = _session(22)
    cos, sin = _tables(rng, 200, D, torch.float32)
    qkv = bf16(rng.standard_normal((3, (HQ + 2 * HKV) * D)))
    plens = ints([prefix])

    def step(lens, pos):
        q = T.paged_rope_cache(qkv, cos, sin, cache.k, cache.v, table, lens, HQ, positions=pos)
        return q, T.shared_prefix_attention(q, cache.k, cache.v, ptable, plens, table, lens), \
            T.paged_attention(q, cache.k, cache.v, table, lens)

    graphs = []
    for first in ([5, 60, 1], [90, 3, 17]):
        lens, pos = ints(first), torch.tensor([prefix + n - 1 for n in first], device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(lens, pos)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(lens, pos)
            lens += 1
            pos += 1
        graphs.append((graph, lens, pos, got, list(first)))
    for _ in range(4):
        for graph, lens, pos, got, now in graphs:
            qkv.copy_(bf16(rng.standard_normal(tuple(qkv.shape))))
            graph.replay()
            torch.cuda.synchronize()
            want = step(ints(now), torch.tensor([prefix + n - 1 for n in now], device=DEV))
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            now[:] = [n + 1 for n in now]
            assert lens.tolist() == now


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_replayed_chunks_follow_the_lengths(kv):
    """A captured call over chunks of prompts, and steps of other sizes that share its workspace."""
    HQ, HKV, D, n = 8, 2, 256, [150, 1, 70]
    rng = np.random.default_rng(28)
    cache = Cache(rng, 200, HKV, 32, D, kv)
    table, starts = cache.table(3, 50), ints(starts_of(n))
    q, one = bf16(rng.standard_normal((221, HQ, D))), bf16(rng.standard_normal((3, HQ, D)))
    scales = {"k_scale": cache.k_scale, "v_scale": cache.v_scale}

    def both(lens):
        return (T.paged_attention(one, cache.k, cache.v, table, lens, **scales),
                T.paged_attention(q, cache.k, cache.v, table, lens, starts, **scales),
                T.shared_prefix_attention(one, cache.k, cache.v, table[2], ints([700]), table[:, :9], lens, **scales)
                if not torch.cuda.is_current_stream_capturing() else None)

    lens = ints([900, 5, 1200])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(lens)
    for now in ([900, 5, 1200], [1600, 700, 71], [150, 0, 1], [1599, 1, 1000]):
        lens.copy_(ints(now))
        graph.replay()
        torch.cuda.synchronize()
        want = both(ints(now))
        for a, b in zip(got[:2], want):
            assert torch.equal(a, b)
        again = both(ints(now))
        for a, b in zip(again, want):
            assert torch.equal(a, b)


def test_streams_at_once():
    """Calls that overlap on two streams, many times over the same inputs."""
    rng = np.random.default_rng(23)
    HQ, HKV, D = 16, 4, 128
    cache = Cache(rng, 400, HKV, 16, D)
    table, lens = cache.table(4, 90), ints([1400, 7, 900, 1201])
    q = [bf16(rng.standard_normal((4, HQ, D))) for _ in range(2)]
    want = [T.paged_attention(x, cache.k, cache.v, table, lens) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(T.paged_attention(q[i], cache.k, cache.v, table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g, want[i])


def test_same_results_every_time():
    """No sum depends on an order that changes from run to run."""
    rng = np.random.default_rng(24)
    cache = Cache(rng, 300, 2, 16, 128)
    table, ptable = cache.table(8, 20), cache.table(1, 60)
    q, lens = bf16(rng.standard_normal((8, 8, 128))), ints(rng.integers(0, 320, 8))
    f = lambda: T.shared_prefix_attention(q, cache.k, cache.v, ptable, ints([950]), table, lens)  # noqa: E731
    want = f()
    for _ in range(10):
        assert torch.equal(f(), want)


def test_inputs_of_other_strides():
    """Rows that begin anywhere: views of wider tensors, odd offsets, transposed heads."""
    rng = np.random.default_rng(25)
    HQ, HKV, D = 4, 2, 64
    cache = Cache(rng, 12, HKV, 16, D)
    table, lens = cache.table(3, 3), ints([40, 7, 48])
    q = bf16(rng.standard_normal((3, HQ, D)))
    want = T.paged_attention(q, cache.k, cache.v, table, lens)
    wide = torch.zeros(3, HQ * D + 11, device=DEV, dtype=BF16)
    wide[:, 3:3 + HQ * D] = q.view(3, -1)
    for x in (wide[:, 3:3 + HQ * D].unflatten(1, (HQ, D)), q.transpose(0, 1).contiguous().transpose(0, 1),
              q.permute(0, 2, 1).contiguous().permute(0, 2, 1)):
        assert torch.equal(T.paged_attention(x, cache.k, cache.v, table, lens), want)
    into = torch.zeros(3, HQ * D + 8, device=DEV, dtype=BF16)
    T.paged_attention(q, cache.k, cache.v, table, lens, out=into[:, 8:])
    assert torch.equal(into[:, 8:], want) and not into[:, :8].any()

    cos, sin = _tables(rng, 50, D, torch.float32)
    qkv = bf16(rng.standard_normal((3, (HQ + 2 * HKV) * D)))
    ref = T.paged_rope_cache(qkv, cos, sin, cache.k, cache.v, table, lens, HQ)
    keys = cache.k.clone()
    odd = torch.zeros(3, qkv.shape[1] + 5, device=DEV, dtype=BF16)
    odd[:, 5:] = qkv
    cs = torch.zeros(2, 50, D + 3, device=DEV)
    cs[0, :, 1:D + 1], cs[1, :, 1:D + 1] = cos, sin
    got = T.paged_rope_cache(odd[:, 5:], cs[0, :, 1:D + 1], cs[1, :, 1:D + 1], cache.k, cache.v, table, lens, HQ)
    assert torch.equal(got, ref) and torch.equal(cache.k, keys)


def test_chunks_between_other_columns():
    """Queries and results that are columns of wider tensors; what lies beside them stays."""
    rng = np.random.default_rng(33)
    HQ, HKV, D, n = 8, 2, 128, [150, 3]
    cache = Cache(rng, 60, HKV, 32, D)
    table, lens, starts = cache.table(2, 30), [900, 77], starts_of(n)
    wide = bf16(rng.standard_normal((153, 3 * HQ, D)))
    big = bf16(rng.standard_normal((155, HQ * D + 64)))
    old = big.clone()
    q, out = wide[:, HQ:2 * HQ], big[1:154, 8:8 + HQ * D]
    assert T.paged_attention(q, cache.k, cache.v, table, ints(lens), ints(starts), out=out) is out
    check_attention(out, q, cache, table, lens, starts)
    out.copy_(old[1:154, 8:8 + HQ * D])
    assert torch.equal(big, old)


def test_nothing_to_do():
    cache = Cache(np.random.default_rng(26), 2, 2, 16, 64)
    none = torch.empty(0, 4, 64, device=DEV, dtype=BF16)
    table, lens = torch.empty(0, 1, device=DEV, dtype=torch.int32), torch.empty(0, device=DEV, dtype=torch.int32)
    assert T.paged_attention(none, cache.k, cache.v, table, lens).shape == (0, 256)
    # sequences without rows
    assert T.paged_attention(none, cache.k, cache.v, ints([[0]]), ints([3]), ints([0, 0])).shape == (0, 256)
    cos, sin = _tables(np.random.default_rng(27), 4, 64, torch.float32)
    q = T.paged_rope_cache(torch.empty(0, 8 * 64, device=DEV, dtype=BF16), cos, sin, cache.k, cache.v, ints([[0]]),
                           ints([3]), 4, ints([0, 0]))
    assert q.shape == (0, 4, 64)


def test_threads_on_one_stream():
    """Calls of two launches each from several host threads on one stream: what each gives when it is alone."""
    rng = np.random.default_rng(34)
    HQ, HKV, D, B = 8, 2, 128, 40
    cache = Cache(rng, 250, HKV, 32, D)
    table, ptable, lens = cache.table(B, 4), cache.table(1, 40), ints(rng.integers(1, 128, B))
    q = [bf16(rng.standard_normal((B, HQ, D))) for _ in range(3)]
    plens = [ints([n]) for n in (1280, 900, 333)]

    def call(i):
        return T.shared_prefix_attention(q[i], cache.k, cache.v, ptable, plens[i], table, lens)

    want = [call(i) for i in range(3)]
    torch.cuda.synchronize()
    got = [[] for _ in range(3)]
    threads = [threading.Thread(target=lambda i=i: got[i].extend(call(i) for _ in range(40))) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(3):
        assert len(got[i]) == 40 and all(torch.equal(g, want[i]) for g in got[i])


def _scales(cache, table):
    """Heads whose codes stand for their negatives, for nothing, and for next to nothing."""
    for scale in (cache.k_scale, cache.v_scale):
        scale[0] = 0.0
        scale[1] *= -1
        scale[2] = 1e-42
    cache.v_scale.copy_(cache.v_scale.roll(1))


@pytest.mark.parametrize("scale", [None, 3.0])
@pytest.mark.parametrize("HQ,HKV,D,n", [(16, 4, 128, None), (8, 4, 64, [5, 9, 3, 2, 7]), (4, 4, 128, [150, 9, 60, 40, 3]),
                                        (16, 4, 64, [80, 9, 40, 5, 0]), (8, 4, 256, [70, 30, 5, 40, 1]),
                                        (16, 4, 256, None)])
def test_attend_any_scale_of_a_head(HQ, HKV, D, n, scale):
    """A head's scale may be negative, zero or tiny: its scores are what codes times scale give."""
    lens = [40, 3, 700, 900, 0]
    _attend(35, HQ, HKV, D, lens, n=n, kv="e4m3", ps=32, edit=_scales, scale=scale)
    _attend(36, HQ, HKV, D, lens, n=n, kv="e4m3", ps=32, edit=_scales, scale=scale, prefix=([300, 33], [0, 3, 4]))


@pytest.mark.parametrize("D,rows", [(128, 3), (64, 100), (256, 100)])
def test_attend_a_scale_that_is_no_number(D, rows):
    """What such a head's rows attend is NaN, a row that attends nothing zero, the other head as without it."""
    cache = Cache(np.random.default_rng(37), 10, 2, 32, D, "e4m3")
    table, q = cache.table(2, 4), bf16(np.random.default_rng(38).standard_normal((2 * rows, 4, D)))
    lens, starts = ints([rows - 2, 0]), ints([0, rows, 2 * rows])
    f = lambda: T.paged_attention(q, cache.k, cache.v, table, lens, starts, k_scale=cache.k_scale,  # noqa: E731
                                  v_scale=cache.v_scale).view(2 * rows, 2, 2 * D)
    want = f()
    cache.k_scale[0] = float("nan")
    got = f()
    assert torch.isnan(got[2:rows, 0]).all() and not got[:2].any() and not got[rows:].any()
    assert torch.equal(got[:, 1], want[:, 1])


FEW = [(16, 8, 128, None), (16, 1, 128, None), (6, 2, 64, None), (16, 4, 256, None), (8, 2, 128, [5, 5, 5, 5]),
       (4, 2, 64, [9, 2, 12, 1]), (8, 2, 256, [4, 4, 3, 4])]


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D,n", FEW)
def test_few_rows_keep_their_probabilities(HQ, HKV, D, n, kv):
    """Two bf16 parts of each, in chunks that are joined and with a prefix too."""
    rng = np.random.default_rng(39)
    cache, lens = Cache(rng, 120, HKV, 32, D, kv), [290, 40, 17, 500]
    table, ptable, plens = cache.table(4, 16), cache.table(1, 10), [277]
    starts = None if n is None else starts_of(n)
    q = bf16(rng.standard_normal((4 if n is None else sum(n), HQ, D)) * 1.5)
    args = (table, ints(lens), None if n is None else ints(starts))
    scales = {"k_scale": cache.k_scale, "v_scale": cache.v_scale}
    check_parts(T.paged_attention(q, cache.k, cache.v, *args, **scales), q, cache, table, lens, starts)
    if sum(n or [1] * 4) * HQ // HKV <= (16 if D == 256 else 32):  # (all rows are the prefix's)
        got = T.shared_prefix_attention(q, cache.k, cache.v, ptable, ints(plens), *args, **scales)
        check_parts(got, q, cache, table, lens, starts, None, (ptable.cpu().numpy(), plens, None))


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D,rows", [(4, 2, 64, 1), (16, 1, 128, 2), (16, 4, 256, 1), (4, 2, 128, 9)])
def test_few_rows_do_not_round_their_probabilities_to_bf16(HQ, HKV, D, rows, kv):
    """Probabilities midway between two bf16 numbers; the earlier rows of several attend fewer of them."""
    cache = Cache(np.random.default_rng(40), 8, HKV, 16, D, kv)
    table = cache.table(1, 7)
    for scale in (cache.k_scale, cache.v_scale):
        if scale is not None:
            scale.fill_(1.0)
    scale = midway(cache, table)
    q = torch.zeros(rows, HQ, D, device=DEV, dtype=BF16)
    q[:, :, 0] = 1.0
    got = T.paged_attention(q, cache.k, cache.v, table, ints([KEYS]), ints([0, rows]), scale=scale, k_scale=cache.k_scale,
                            v_scale=cache.v_scale)
    check_parts(got, q, cache, table, [KEYS], [0, rows], scale)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", [(8, 2, 256), (4, 4, 256), (8, 2, 128), (16, 1, 64), (6, 2, 64)])
def test_prefix_prompts(HQ, HKV, D, kv):
    """Prompts and chunks behind prefixes, their own keys cut too: tiles of 64 and 128 rows with a launch that joins
    their parts; sequences of no prefix, of no rows, of no own positions for some rows."""
    _attend(41, HQ, HKV, D, [150, 1, 0, 700, 5, 40], n=[150, 1, 0, 70, 5, 44], kv=kv, ps=32,
            prefix=([600, 33], [0, 4, 5]), before=1, behind=2)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("HQ,HKV,D", [(16, 4, 256), (8, 2, 128), (4, 4, 64)])
def test_prefix_drafted_tokens_of_many(HQ, HKV, D, kv):
    """A few rows for each of many sequences: a prefix's tiles hold rows of several sequences."""
    rng = np.random.default_rng(42)
    _attend(42, HQ, HKV, D, list(rng.integers(2, 300, 20)), n=rng.integers(0, 6, 20), kv=kv, ps=32,
            prefix=([900, 100, 257], [0, 9, 9, 18]))


def test_append_by_a_scale_of_zero():
    """value / 0: the largest code of either sign, NaN for a value of 0."""
    cache = Cache(np.random.default_rng(43), 2, 1, 16, 64, "e4m3")
    cache.v_scale.zero_()
    x = torch.zeros(1, 3 * 64, device=DEV, dtype=BF16)
    x[0, 128:130] = torch.tensor([1e-3, -2.0])
    one, zero = torch.ones(1, 64, device=DEV), torch.zeros(1, 64, device=DEV)
    T.paged_rope_cache(x, one, zero, cache.k, cache.v, ints([[1]]), ints([1]), 1, k_scale=cache.k_scale,
                       v_scale=cache.v_scale)
    v = cache.v.float()[1, 0, 0]
    assert v[:2].tolist() == [448.0, -448.0] and torch.isnan(v[2:]).all()


@pytest.mark.parametrize("HQ,HKV,D,rows", [(4, 4, 128, 5), (4, 4, 128, 150), (8, 4, 64, 60), (8, 4, 256, 70)])
def test_later_rows_have_no_part_whatever_the_scales(HQ, HKV, D, rows):
    """A value that is NaN in the last token, with scales of any sign and zero: the rows before it are as without it."""
    rng = np.random.default_rng(44)
    cache = Cache(rng, 20, HKV, 32, D, "e4m3")
    table = cache.table(1, 16)
    _scales(cache, table)
    q, j = bf16(rng.standard_normal((rows, HQ, D))), rows + 330
    cache.v.view(torch.uint8)[int(table[0, j // 32]), :, j % 32, ::3] = 0x7F
    out = T.paged_attention(q, cache.k, cache.v, table, ints([j + 1]), ints([0, rows]), k_scale=cache.k_scale,
                            v_scale=cache.v_scale)
    check_attention(out[:-1], q[:-1], cache, table, [j], [0, rows - 1])
    assert torch.isnan(out[-1].view(HQ, D)[:, ::3]).all()
