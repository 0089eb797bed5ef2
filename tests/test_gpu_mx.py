"""Operators over microscaled blocks on the GPU, against the oracle in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from torch import nn

from oracle import bz_mx_oracle as O
from tests._util import bf16_tensor

from breeze_amd import _lib as L
from breeze_amd import gemv as G
from breeze_amd import mx
from breeze_amd import mxfp4_linear as M4
from breeze_amd import quantized_checkpoint as Q
from breeze_amd.fused import kernels as FK

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ELEMS = [O.E2M1, O.E4M3]


def _np(t):
    return t.detach().double().cpu().numpy()


def _rows(m, k, seed=0, dtype=BF16, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(spread * torch.randn(k, generator=g))
    return x.to(dtype).cuda()


def _codes(codes, elem):
    """The GPU's codes as one element code a byte."""
    c = codes.view(torch.uint8).cpu().numpy()
    return np.stack([c & 15, c >> 4], -1).reshape(c.shape[0], -1) if elem == O.E2M1 else c


class Weight:
    """A random e2m1 weight: oracle codes, values and the GPU's buffers."""

    def __init__(self, n, k, seed=0, paired=False):
        rng = np.random.default_rng(seed + n + k)
        w = rng.standard_normal((n, k)) * k ** -0.5 * np.exp(rng.standard_normal((n, 1)))
        self.n, self.k = n, k
        self.codes, self.scales = O.quantize(w, O.E2M1)
        self.values = O.values(self.codes, self.scales, O.E2M1)
        self.rows = torch.from_numpy(O.pack_nibbles(self.codes)).cuda()
        self.sc = torch.from_numpy(self.scales).cuda()
        self.fmt = G.W_MXFP4_TILED_PAIRED if paired else G.W_MXFP4_TILED
        self.tiled = torch.from_numpy(O.tile(self.codes, self.scales, O.E2M1, paired)).cuda()


def _bound(x, w, ref, k, out_dtype=BF16, before=0.0, extra=0.0):
    """Rounding of the output, and of K fp32 additions (2^-24 of the sum of
    magnitudes each); before: relative error of the product before the
    epilogue, extra: absolute."""
    total = np.abs(x) @ np.abs(w).T
    return torch.finfo(out_dtype).eps / 2 * (np.abs(ref) + extra) + (k * 2.0 ** -24 + before) * total + extra


def _close(out, ref, bound):
    err = np.abs(_np(out) - ref)
    assert (err <= bound).all(), (err / np.maximum(bound, 1e-300)).max()


# ---- quantising and reading back ---------------------------------------------------------------------


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k", [(1, 32), (3, 96), (17, 160), (2, 2560), (301, 672)])
def test_quantize(elem, dtype, m, k):
    x = _rows(m, k, 1, dtype, 2.0)
    codes, scales = mx.quantize_mx(x, elem)
    want, want_s = O.quantize(_np(x), elem)
    assert (_codes(codes, elem) == want).all() and (scales.cpu().numpy() == want_s).all()
    for dt in (BF16, F32):
        got = mx.dequantize_mx(codes, scales, elem, dt)
        assert got.dtype == dt and (_np(got) == O.values(want, want_s, elem)).all()


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_quantize_strides_and_alignment(elem, dtype):
    base = _rows(9, 700, 2, dtype)
    views = [base[:, 1:577], base[:, 8:584], base[::2, 3:35], base.t()[:96, :5].t(), base[4:5].expand(6, 700)[:, :32],
             base.view(-1)[1:1 + 640].view(5, 128)]
    for x in views:
        codes, scales = mx.quantize_mx(x, elem)
        want, want_s = O.quantize(_np(x), elem)
        assert (_codes(codes, elem) == want).all() and (scales.cpu().numpy() == want_s).all()
    x = views[1][:, :512]
    got, (c, s) = mx.mx_rows(x, elem), O.quantize(_np(x), elem)
    assert (got.data.cpu().numpy() == O.tile(c, s, elem)).all()
    x = views[0][:, :512]  # rows at odd addresses
    got, (c, s) = mx.mx_rows(x, elem), O.quantize(_np(x), elem)
    assert (got.data.cpu().numpy() == O.tile(c, s, elem)).all()


@pytest.mark.parametrize("elem", ELEMS)
def test_every_bf16_value_rounds_to_nearest_even(elem):
    """Each magnitude in a block of its own beside the block's largest."""
    bits = np.arange(0x7F80, dtype=np.uint16)
    for top in (0x4000, 0x3F80, 0x0080, 0x0001, 0x7F7F, 0x3FC0):
        x = np.zeros((bits.size, 32), np.uint16)
        x[:, 0], x[:, 1], x[:, 2] = top, bits, bits | 0x8000
        x = bf16_tensor(x)
        codes, scales = mx.quantize_mx(x, elem)
        want, want_s = O.quantize(_np(x), elem)
        assert (_codes(codes, elem) == want).all() and (scales.cpu().numpy() == want_s).all()


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_blocks_with_nan_infinity_zero_and_the_extremes(elem, dtype):
    fi = torch.finfo(dtype)
    x = torch.zeros(8, 256, dtype=dtype)
    x[0, 5], x[1, 37], x[2, 64], x[3, 255] = float("nan"), float("inf"), -float("inf"), -float("nan")
    x[4] = -0.0
    x[5, :64], x[5, 64:] = fi.max, -fi.max
    x[6, ::3], x[6, 1::3] = fi.tiny, -fi.tiny / 4
    x[7] = torch.randn(256).to(dtype)
    x[0, 64:], x[1, :32] = 1.5, 2.5
    x = x.cuda()
    codes, scales = mx.quantize_mx(x, elem)
    want, want_s = O.quantize(_np(x), elem)
    assert (scales.cpu().numpy() == want_s).all()
    keep = np.repeat(want_s != 255, 32, -1)
    assert (_codes(codes, elem) == want)[keep].all()
    assert [(want_s[i] == 255).sum() for i in range(8)] == [1, 1, 1, 1, 0, 0, 0, 0]
    for dt in (BF16, F32):
        got = _np(mx.dequantize_mx(codes, scales, elem, dt))
        assert (np.isnan(got) == ~keep).all() and (got == O.values(want, want_s, elem))[keep].all()


@pytest.mark.parametrize("elem", ELEMS)
def test_read_back_every_code_and_scale(elem):
    n = 16 if elem == O.E2M1 else 256
    codes = np.tile(np.arange(n, dtype=np.uint8), (256, 256 // n))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 8, 1)
    want = O.values(codes, scales, elem)
    if elem == O.E4M3:
        want[:, [127, 255]] = np.nan  # the type's own NaN
    dev = torch.from_numpy(O.pack_nibbles(codes) if elem == O.E2M1 else codes).cuda()
    got = mx.dequantize_mx(dev, torch.from_numpy(scales).cuda(), elem, F32)
    with np.errstate(over="ignore"):
        assert np.array_equal(_np(got), want.astype(np.float32).astype(np.float64), equal_nan=True)
    got = mx.dequantize_mx(dev, torch.from_numpy(scales).cuda(), elem)
    fits = torch.from_numpy(want).to(BF16)  # exact but below 2^-126 and above the range
    assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=7e37), torch.nan_to_num(fits.float(), nan=7e37))


def test_read_back_of_other_layouts():
    x = _rows(6, 128, 3)
    codes, scales = mx.quantize_mx(x)
    want = mx.dequantize_mx(codes, scales)
    buf = torch.zeros(6 * 64 + 1, dtype=torch.uint8, device="cuda")
    buf[1:].view(6, 64).copy_(codes)
    assert torch.equal(mx.dequantize_mx(buf[1:].view(6, 64), scales.t().contiguous().t()), want)
    assert torch.equal(mx.dequantize_mx(codes[::2], scales[::2]), want[::2])
    with pytest.raises(ValueError, match="not those of"):
        mx.dequantize_mx(codes, scales[:, :3])
    with pytest.raises(ValueError, match="not those of"):
        mx.dequantize_mx(codes, scales, "e4m3")
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        mx.dequantize_mx(codes, scales, dtype=F16)


def test_quantize_refusals_and_no_rows():
    x = _rows(4, 128)
    for bad, err in ((x[:, :40], ValueError), (x[:, :0], ValueError), (x[0], ValueError), (x.double(), TypeError)):
        with pytest.raises(err):
            mx.quantize_mx(bad)
    with pytest.raises(ValueError, match="multiple of 128"):
        mx.mx_rows(x[:, :96])
    with pytest.raises(RuntimeError, match="no gradient"):
        mx.mx_rows(x.float().requires_grad_())
    c, s = mx.quantize_mx(x[:0])
    assert c.shape == (0, 64) and s.shape == (0, 4) and mx.dequantize_mx(c, s).shape == (0, 128)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("m,k", [(1, 128), (16, 384), (17, 512), (33, 640), (130, 1280)])
def test_tiled_rows(elem, m, k):
    for dtype in (BF16, F16, F32):
        x = _rows(m, k, 4, dtype)
        got = mx.mx_rows(x, elem)
        assert got.shape == (m, k) and (got.data.cpu().numpy() == O.tile(*O.quantize(_np(x), elem), elem)).all()


# ---- the weight's layouts ------------------------------------------------------------------------------


@pytest.mark.parametrize("n,k", [(16, 128), (48, 640), (160, 1280)])
@pytest.mark.parametrize("paired", [False, True])
def test_packing(n, k, paired):
    w = Weight(n, k, paired=paired)
    got = G.pack_tiled(G.W_MXFP4, w.rows, k, w.fmt, sc0=w.sc)
    assert torch.equal(got, w.tiled)
    assert (_np(G.dequant(w.fmt, got, n, k)) == w.values).all()
    assert (_np(G.dequant(G.W_MXFP4, w.rows, n, k, sc0=w.sc)) == w.values).all()
    plain = torch.from_numpy(O.tile(w.codes, w.scales, O.E2M1)).cuda()
    assert torch.equal(G.pack_tiled(G.W_MXFP4_TILED, plain, k, w.fmt), w.tiled)
    if n % 32 == 0 and n > 32:  # by halves: gate, then up
        out = None
        for i, r in enumerate(torch.split(w.rows, n // 2)):
            out = G.pack_tiled(G.W_MXFP4, r.contiguous(), k, w.fmt, sc0=w.sc[i * n // 2:(i + 1) * n // 2].contiguous(),
                               n_total=n, row0=i * n // 2, out=out)
        assert torch.equal(out, w.tiled)


# ---- bf16 rows times the weight --------------------------------------------------------------------------


def _gemv_reference(x, w, epi, gamma, eps, res, out_dtype):
    xd, extra, before = _np(x), 0.0, 0.0
    if gamma is not None:
        xd, scale = _np((x.float() * gamma.float()).to(BF16)), O.rmsnorm_scale(xd, eps)
        before = 2.0 ** -20 + x.shape[1] * 2.0 ** -24  # of 1 / rms: K sums, the mean, the root
    else:
        scale = np.ones((x.shape[0], 1))
    y = xd @ w.values.T * scale
    if epi == G.EPI_SILU_GATE:
        h = w.n // 2
        g, u = y[:, :h], y[:, h:]
        ref = O.silu(g) * u
        # d silu <= 1.1 dg; the exponential and the division are within 2^-20 of it
        eg, eu = (_bound(np.abs(xd) * scale, p, 0.0, w.k, before=before) for p in (w.values[:h], w.values[h:]))
        bound = torch.finfo(out_dtype).eps / 2 * np.abs(ref) + (1.1 * eg * np.abs(u) + (np.abs(O.silu(g)) + 1.1 * eg) * eu
                                                                + 2.0 ** -20 * np.abs(ref)) * 1.01
        return ref, bound
    ref = y
    if epi == G.EPI_RESIDUAL:
        ref = y + _np(res)
        extra = 2.0 ** -24 * np.abs(ref)
    return ref, _bound(np.abs(xd) * scale, w.values, ref, w.k, out_dtype, before, extra)


@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 16, 17, 33])
@pytest.mark.parametrize("n,k", [(16, 128), (272, 640), (64, 2048), (4112, 512), (2560, 1280)])
@pytest.mark.parametrize("epi,norm", [(G.EPI_NONE, False), (G.EPI_RESIDUAL, False), (G.EPI_SILU_GATE, True),
                                      (G.EPI_NONE, True), (G.EPI_SILU_GATE, False)])
def test_gemv(m, n, k, epi, norm):
    w = Weight(n, k, paired=epi == G.EPI_SILU_GATE)
    x = _rows(m, k, 5)
    gamma = (1 + 0.2 * torch.randn(k)).to(BF16).cuda() if norm else None
    n_out = n // 2 if epi == G.EPI_SILU_GATE else n
    res = torch.randn(m, n_out).to(BF16).cuda() if epi == G.EPI_RESIDUAL else None
    out = G.gemv(x, w.tiled, w.fmt, n, gamma=gamma, epilogue=epi, residual=res)
    _close(out, *_gemv_reference(x, w, epi, gamma, 1e-6, res, BF16))


@pytest.mark.parametrize("m,n,k", [(1, 2560, 10240), (2, 1024, 10240), (7, 1024, 8192), (13, 1024, 8192), (32, 2560, 10240),
                                   (4, 20480, 2560)])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_gemv_long_rows(m, n, k, out_dtype):
    w, x = Weight(n, k), _rows(m, k, 6)
    res = torch.randn(m, n).to(out_dtype).cuda()
    out = G.gemv(x, w.tiled, w.fmt, n, epilogue=G.EPI_RESIDUAL, residual=res, out_dtype=out_dtype)
    _close(out, *_gemv_reference(x, w, G.EPI_RESIDUAL, None, 0.0, res, out_dtype))


def test_gemv_second_store_strides_and_forced_shapes():
    w = Weight(96, 640)
    wide = torch.randn(5, 700).to(BF16).cuda()
    x = wide[:, 8:648]  # rows at 16-byte steps of 1400 bytes: copied by the wrapper or read in place
    out, out2 = torch.zeros(5, 128, device="cuda", dtype=BF16), torch.zeros(5, 32, device="cuda", dtype=BF16)
    G.gemv(x, w.tiled, w.fmt, 96, out=out[:, 16:112], out2=out2)
    ref, bound = _gemv_reference(x, w, G.EPI_NONE, None, 0.0, None, BF16)
    _close(out[:, 16:112], ref, bound)
    assert torch.equal(out2, out[:, 16:48]) and not out[:, :16].any() and not out[:, 112:].any()
    for cfg in ((0, 0, 0, 5), (0, 3, 0, 5), (0, 0, 1, 5), (0, 2, 3, 5), (0, 1, 8, 5), (0, 0, 0, 6), (0, 2, 4, 6),
                (0, 0, 2, 6, 2)):
        _close(G.gemv(x, w.tiled, w.fmt, 96, cfg=cfg), ref, bound)


@pytest.mark.parametrize("m", [33, 64, 203, 300])
@pytest.mark.parametrize("n,k", [(48, 128), (272, 640), (2560, 1280), (80, 4992)])
def test_prompt(m, n, k):
    w, x = Weight(n, k), _rows(m, k, 7)
    out = G.dequant_matmul(x, w.tiled, w.fmt, n, k)
    _close(out, *_gemv_reference(x, w, G.EPI_NONE, None, 0.0, None, BF16))


def test_prompt_follows_autograd():
    w, x = Weight(48, 256), _rows(40, 256, 8, F32)
    x.requires_grad_()
    g = torch.randn(40, 48).to(BF16).cuda()
    G.dequant_matmul(x, w.tiled, w.fmt, 48, 256).backward(g)
    ref = _np(g) @ w.values
    # the gradient of a bf16 product, rounded once to bf16
    _close(x.grad, ref, 2.0 ** -8 * np.abs(ref) + 48 * 2.0 ** -24 * (np.abs(_np(g)) @ np.abs(w.values)))


# ---- quantised rows times the weight ---------------------------------------------------------------------


def _eights(codes, scales, elem, least):
    """Largest magnitude of each eight consecutive columns, at least ``least``
    times the block's scale."""
    v = np.abs(O.values(codes, scales, elem)).reshape(codes.shape[0], -1, 8).max(-1)
    return np.maximum(v, least * np.repeat(np.ldexp(1.0, scales.astype(np.int64) - 127), 4, -1))


def _mx_reference(x, w, elem, res, out_dtype):
    """With 8-bit elements the matrix core adds eight products (those of eight
    consecutive columns) on a grid: each is cut toward zero at 2^(E - 13), E
    the largest sum of the two factors' exponents among the eight
    (test_the_grid_of_eight_products).  An exponent is that of the magnitude,
    but at least -6 for e4m3 and 0 for e2m1, the types' subnormal ones; so
    2^E <= max(|a|, 2^-6 s_a) max(|b|, s_b) over the eight, with the blocks'
    scales s.  Seven products can lose less than a grid step each (the one
    that sets E spans 4 + 2 bits and loses nothing).  4-bit products lie
    within 2^-6 of one another and lose nothing."""
    codes, scales = O.quantize(_np(x), elem)
    xq = O.values(codes, scales, elem)
    ref, extra = xq @ w.values.T, 0.0
    if elem == O.E4M3:
        extra = 7 * 2.0 ** -13 * (_eights(codes, scales, elem, 2.0 ** -6) @ _eights(w.codes, w.scales, O.E2M1, 1.0).T)
    if res is not None:
        ref = ref + _np(res)
        extra = extra + 2.0 ** -24 * np.abs(ref)
    return ref, _bound(xq, w.values, ref, w.k, out_dtype, extra=extra)


def test_the_grid_of_eight_products():
    """2^10 - 2^10 + 2^e: what the tolerance of 8-bit products rests on."""
    w = Weight(16, 128)
    w.codes[:], w.scales[:] = 0, 127
    for small, lost in ((2, True), (7, True), (8, False), (40, False), (100, False)):
        w.codes[:] = 0
        w.codes[:, 0], w.codes[:, 1], w.codes[:, small] = 6, 14, 2  # 4, -4, 1
        tiled = torch.from_numpy(O.tile(w.codes, w.scales, O.E2M1)).cuda()
        e = np.arange(-9, 9)
        x = np.zeros((e.size, 128))
        x[:, 0] = x[:, 1] = 256
        x[:, 32::32] = 256  # every block's scale is 1; these columns meet zeros
        x[:, small] = 2.0 ** e
        out = mx.mx_linear(mx.mx_rows(torch.from_numpy(x).float().cuda(), O.E4M3), tiled, 16, out_dtype=F32)
        want = np.where(lost & (e < -3), 0.0, 2.0 ** e)
        assert (_np(out) == want[:, None]).all()


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 32, 33, 48, 65, 129, 257, 300])
@pytest.mark.parametrize("n,k", [(16, 128), (48, 384), (272, 640), (528, 1280), (1040, 2176)])
def test_mx_linear(elem, m, n, k):
    w, x = Weight(n, k), _rows(m, k, 9)
    res = torch.randn(m, n).to(BF16).cuda() if (m + n) % 3 else None
    out = mx.mx_linear(x, w.tiled, n, elem=elem, residual=res)
    _close(out, *_mx_reference(x, w, elem, res, BF16))
    assert torch.equal(mx.mx_linear(mx.mx_rows(x, elem), w.tiled, n, residual=res), out) or m <= 32
    again = mx.mx_linear(mx.mx_rows(x, elem), w.tiled, n, residual=res)
    _close(again, *_mx_reference(x, w, elem, res, BF16))


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("m,n,k", [(1, 2560, 10240), (5, 1024, 8192), (40, 2560, 10240), (513, 2560, 2560), (1030, 4096, 1024)])
def test_mx_linear_of_layers(elem, m, n, k):
    w, x = Weight(n, k), _rows(m, k, 10)
    res = torch.randn(m, n).to(F32).cuda()
    out = mx.mx_linear(x, w.tiled, n, elem=elem, residual=res, out_dtype=F32)
    _close(out, *_mx_reference(x, w, elem, res, F32))


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("m", [3, 40, 260])
def test_mx_linear_types_strides_and_aliases(elem, m):
    n, k = 144, 512
    w = Weight(n, k)
    for dtype in (F16, F32):
        x = _rows(m, k, 11, dtype)
        _close(mx.mx_linear(x, w.tiled, n, elem=elem), *_mx_reference(x, w, elem, None, BF16))
    wide = _rows(m, 600, 12)
    for x in (wide[:, 8:520], wide[:, 1:513], wide[:1, 3:515].expand(m, k), wide.t()[7:519].t()):
        _close(mx.mx_linear(x, w.tiled, n, elem=elem), *_mx_reference(x, w, elem, None, BF16))
    # rows of wider tensors, the residual in the output's place, the rest untouched
    x = wide[:, 8:520]
    big = torch.randn(m + 2, n + 40).to(BF16).cuda()
    before, out = big.clone(), big[1:m + 1, 17:17 + n]
    ref, bound = _mx_reference(x, w, elem, out.clone(), BF16)
    assert mx.mx_linear(x, w.tiled, n, elem=elem, residual=out, out=out) is out
    _close(out, ref, bound)
    before[1:m + 1, 17:17 + n] = big[1:m + 1, 17:17 + n]
    assert torch.equal(before, big)
    # a residual that lies partly in the output
    flat = torch.randn(2 * m * n).to(BF16).cuda()
    out, res = flat[:m * n].view(m, n), flat[5:5 + m * n].view(m, n)
    ref, bound = _mx_reference(x, w, elem, res.clone(), BF16)
    _close(mx.mx_linear(x, w.tiled, n, elem=elem, residual=res, out=out), ref, bound)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("m", [4, 70])
def test_mx_linear_rows_with_nan_and_infinity(elem, m):
    """Rows are independent: those with a block that cannot be quantised are NaN, the others as ever."""
    n, k = 48, 640
    w, x = Weight(n, k), _rows(m, k, 13)
    clean = mx.mx_linear(x, w.tiled, n, elem=elem)
    x[1, 300], x[3, 0] = float("nan"), float("inf")
    out = mx.mx_linear(x, w.tiled, n, elem=elem)
    bad = torch.zeros(m, dtype=torch.bool)
    bad[1] = bad[3] = True
    assert out[bad.cuda()].isnan().all() and torch.equal(out[~bad.cuda()], clean[~bad.cuda()])


@pytest.mark.parametrize("elem", ELEMS)
def test_mx_linear_large_and_small_scales(elem):
    """Blocks from 2^-60 to 2^60 in one row: each scale stays its own."""
    n, k, m = 32, 512, 40
    w = Weight(n, k)
    x = (_rows(m, k, 14, F32) * 2.0 ** torch.linspace(-60, 60, 16).round().repeat_interleave(32).cuda()).to(BF16)
    _close(mx.mx_linear(x, w.tiled, n, elem=elem, out_dtype=F32), *_mx_reference(x, w, elem, None, F32))


def test_mx_linear_refusals():
    w, x = Weight(32, 256), _rows(4, 256)
    for kw, err in (({"elem": "int4"}, ValueError), ({"residual": x}, ValueError), ({"out_dtype": F16}, TypeError),
                    ({"out": torch.empty(4, 32, device="cuda", dtype=F16)}, ValueError),
                    ({"out": torch.empty(32, 4, device="cuda", dtype=BF16).t()}, ValueError),
                    ({"out": torch.empty(1, 32, device="cuda", dtype=BF16).expand(4, 32)}, ValueError),
                    ({"out": x[:, :32]}, ValueError), ({"residual": torch.zeros(4, 32)}, RuntimeError)):
        with pytest.raises(err):
            mx.mx_linear(x, w.tiled, 32, **kw)
    for bad in (w.tiled[:-16], w.tiled.view(2, -1).t(), torch.cat([w.tiled, w.tiled])):
        with pytest.raises(ValueError, match="W_MXFP4_TILED"):
            mx.mx_linear(x, bad, 32)
    with pytest.raises(ValueError, match="W_MXFP4_TILED"):
        mx.mx_linear(x, w.tiled, 24)
    with pytest.raises(ValueError, match="multiple of 128"):
        mx.mx_linear(x[:, :192], w.tiled, 32)
    with pytest.raises(RuntimeError, match="no gradient"):
        mx.mx_linear(x.float().requires_grad_(), w.tiled, 32)
    assert mx.mx_linear(x[:0], w.tiled, 32).shape == (0, 32)
    assert mx.mx_linear(mx.mx_rows(x[:0]), w.tiled, 32).shape == (0, 32)


@pytest.mark.parametrize("m", [2, 20, 150])
def test_runs_in_a_graph_and_on_another_stream(m):
    """Several operators in a row, captured, replayed beside eager work on new inputs."""
    n, k = 96, 640
    w, w2 = Weight(n, k), Weight(k, 128 * 3, seed=1)
    x, g = _rows(m, k, 15), (1 + 0.1 * torch.randn(k)).to(BF16).cuda()
    src = _rows(m, 384, 16)

    def run():
        h = mx.mx_linear(src, w2.tiled, k, elem="e4m3", residual=x)
        codes, scales = mx.quantize_mx(h, "e2m1")
        q = mx.mx_rows(h, "e2m1")
        a = mx.mx_linear(q, w.tiled, n)
        b = G.gemv(h, w.tiled, w.fmt, n, gamma=g)
        return mx.dequantize_mx(codes, scales), a, b, mx.mx_linear(h, w.tiled, n, elem="e4m3", residual=a)

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(4):
        x.copy_(_rows(m, k, 20 + i))
        src.copy_(_rows(m, 384, 30 + i))
        graph.replay()
        eager = run()
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, eager):
        assert torch.equal(a, b)


# ---- the module --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("n,k", [(64, 256), (50, 200)])
@pytest.mark.parametrize("act_bits", [16, 8, 4])
def test_module(n, k, act_bits):
    lin = nn.Linear(k, n, bias=False).cuda()
    mod = M4.Mxfp4Linear(lin, act_bits=act_bits)
    wq = O.rounded(np.pad(_np(lin.weight), ((0, 0), (0, -k % 32))), O.E2M1)[:, :k]
    for shape in ((3, k), (1, k), (2, 30, k), (4, 5, 9, k)):
        x = torch.randn(*shape).to(BF16).cuda()
        xd = _np(x).reshape(-1, k)
        if xd.shape[0] > M4.PREFILL_ROWS and act_bits != 16:
            xd = O.rounded(np.pad(xd, ((0, 0), (0, -k % 32))), {8: O.E4M3, 4: O.E2M1}[act_bits])[:, :k]
        with torch.no_grad():
            out = mod(x)
        assert out.shape == (*shape[:-1], n) and out.dtype == BF16
        ref = xd @ wq.T
        _close(out.reshape(-1, n), ref, _bound(xd, wq, ref, k))
    assert mod(torch.randn(3, k).cuda()).dtype == F32
    assert mod(torch.zeros(0, k, device="cuda", dtype=BF16)).shape == (0, n)
    cpu = M4.Mxfp4Linear(nn.Linear(k, n, bias=False), device="cuda")
    assert cpu.weight_mxfp4.is_cuda


def test_module_gradient_of_a_prompt():
    lin = nn.Linear(256, 48, bias=False).cuda()
    x = torch.randn(40, 256, device="cuda", requires_grad=True)
    M4.Mxfp4Linear(lin)(x).sum().backward()
    ref = np.ones((40, 48)) @ O.rounded(_np(lin.weight), O.E2M1)
    _close(x.grad, ref, 2.0 ** -8 * np.abs(ref) + 48 * 2.0 ** -24 * 48 * np.abs(O.rounded(_np(lin.weight), O.E2M1)).max())
    with pytest.raises(RuntimeError, match="no gradient"):
        M4.Mxfp4Linear(lin, act_bits=8)(x)


def test_module_swap_checkpoint_and_compile(tmp_path):
    class Mlp(nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj, self.up_proj = (nn.Linear(256, 512, bias=False) for _ in range(2))
            self.down_proj = nn.Linear(512, 256, bias=False)

        def forward(self, x):
            return self.down_proj(torch.nn.functional.silu(self.gate_proj(x)) * self.up_proj(x))

    mlp = Mlp().cuda().to(BF16)
    stats = M4.quantize_module_mxfp4(mlp, min_bytes=0, act_bits=8)
    assert stats == {"converted": 3, "skipped_below_threshold": 0, "weight_bytes_saved": 3 * 262144 * 47 // 64}
    x = torch.randn(5, 256).to(BF16).cuda()
    with torch.no_grad():
        want = mlp(x)
        Q.save_quantized(mlp, tmp_path, {}, source="synthetic")
        fresh = Mlp()
        Q.install_shells(fresh, Q.read_manifest(tmp_path), "cuda")
        Q.load_quantized_state(fresh, tmp_path, "cuda")
        assert torch.equal(fresh(x), want) and fresh.up_proj.act_bits == 8
        assert torch.equal(torch.compile(mlp.up_proj, fullgraph=True, backend="eager")(x), mlp.up_proj(x))


def test_fused_weight_of_modules():
    """gate|up of a SiLU-gate MLP as one launch, behind the norm."""
    gate, up, down = (M4.Mxfp4Linear(nn.Linear(a, b, bias=False).cuda()) for a, b in ((256, 512), (256, 512), (512, 256)))
    x, g = _rows(2, 256, 17), (1 + 0.1 * torch.randn(256)).to(BF16).cuda()
    wgu, wd = FK.FusedWeight.from_mxfp4(gate, up, paired=True), FK.FusedWeight.from_mxfp4(down)
    assert (wgu.N, wgu.K, wgu.layout, wd.layout) == (1024, 256, "mx-tiled-paired", "mx-tiled")
    act = FK.rms_gemv(x, wgu, g, epilogue=G.EPI_SILU_GATE)
    out = FK.rms_gemv(act, wd, None, epilogue=G.EPI_RESIDUAL, residual=x)
    w = Weight.__new__(Weight)
    w.n, w.k = 1024, 256
    w.values = np.concatenate([_np(G.dequant(G.W_MXFP4_TILED, m.weight_mxfp4, 512, 256)) for m in (gate, up)])
    _close(act, *_gemv_reference(x, w, G.EPI_SILU_GATE, g, 1e-6, None, BF16))
    w.n, w.k, w.values = 256, 512, _np(G.dequant(G.W_MXFP4_TILED, down.weight_mxfp4, 256, 512))
    _close(out, *_gemv_reference(act, w, G.EPI_RESIDUAL, None, 0.0, x, BF16))
    assert torch.equal(FK.rms_gemv(act, wd.clone(), None), FK.rms_gemv(act, wd, None))
    with pytest.raises(ValueError, match="paired"):
        FK.rms_gemv(x, wgu, g)
    unpaired = FK.FusedWeight.from_mxfp4(gate, up)
    gu = FK.rms_gemv(x, unpaired, g)
    two = FK.rms_gemv(x, unpaired, g, epilogue=G.EPI_SILU_GATE)
    assert torch.equal(two, FK.silu_mul(gu[:, :512], gu[:, 512:]))


def test_fused_layer_of_modules():
    """A decoder layer whose seven projections are Mxfp4Linear, step by step
    against the float32 layer with the dequantised weights (the bar of
    tests/test_gpu_layer.py)."""
    import copy

    from breeze_amd.fused.layer import FusedDecoderLayer
    from tests.test_gpu_layer import TOL, _cfg, _layer, _run_steps

    cfg = _cfg()
    layer = _layer(cfg)
    ref, own = copy.deepcopy(layer), copy.deepcopy(layer).to("cuda", BF16)
    names = ("gate_proj", "up_proj", "down_proj", "q_proj", "k_proj", "v_proj", "o_proj")
    assert M4.quantize_module_mxfp4(own, target_names=names, min_bytes=0, act_bits=8)["converted"] == 7
    for name, lin in ref.named_modules():
        if name.rpartition(".")[2] in names:
            with torch.no_grad():
                lin.weight.copy_(torch.from_numpy(O.rounded(lin.weight.double().numpy(), O.E2M1)).float())
    errs, c_ref, c_own = _run_steps(cfg, ref, FusedDecoderLayer(own, 0), B=2, S=64, steps=8)
    assert max(errs) <= TOL, errs


# ---- calls beside each other, and what earlier calls leave behind -------------------------------------------


@pytest.mark.parametrize("m", [1, 9, 33])
@pytest.mark.parametrize("k", [128, 384, 640])
def test_packing_into_a_used_buffer(m, k):
    """Rows whose last units do not fill a dword of scale codes: what the buffer held is not read."""
    w, x = Weight(48, k), _rows(m, k, 18)
    used = torch.full_like(w.tiled, 255)
    G.pack_tiled(G.W_MXFP4, w.rows, k, w.fmt, sc0=w.sc, out=used)
    assert torch.equal(used, w.tiled)
    again = torch.full_like(used, 255)
    G.pack_tiled(G.W_MXFP4_TILED, used, k, w.fmt, out=again)
    assert torch.equal(again, w.tiled)
    _close((G.gemv if m <= 32 else lambda x, w, f, n: G.dequant_matmul(x, w, f, n, k))(x, used, w.fmt, 48),
           *_gemv_reference(x, w, G.EPI_NONE, None, 0.0, None, BF16))


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("m", [40, 300])
def test_short_rows_after_rows_of_nan(elem, m):
    """LDS holds codes of NaN from the call before; units past a short row are zeros all the same."""
    bad = torch.full((m, 1024), float("nan"), device="cuda", dtype=BF16)
    wide = Weight(1024, 1024)
    for k in (128, 256, 384, 640):
        w, x = Weight(1024, k), _rows(m, k, 19)
        assert mx.mx_linear(bad, wide.tiled, 1024, elem=elem).isnan().all()
        _close(mx.mx_linear(x, w.tiled, 1024, elem=elem), *_mx_reference(x, w, elem, None, BF16))


def test_forced_shapes():
    """Every launch shape that is built, and refusals of those that are not."""
    n, k = 272, 1664
    w = Weight(n, k)
    for elem in ELEMS:
        for m in (5, 32):
            x = _rows(m, k, 21)
            ref, bound = _mx_reference(x, w, elem, None, BF16)
            for t in (1, 2, 3, 8):
                for upw, nsl in ((0, 0), (0, 3), (1, 2), (2, 1), (3, 1), (4, 2), (5, 1), (5, 13)):
                    _close(mx.mx_linear(x, w.tiled, n, elem=elem, cfg=t | upw << 8 | nsl << 16), ref, bound)
        x = _rows(150, k, 22)
        ref, bound = _mx_reference(x, w, elem, None, BF16)
        for a, b in ((1, 2), (2, 2), (4, 2), (6, 2), (4, 4), (8, 4) if elem == O.E2M1 else (6, 4)):
            for nsl in (0, 1, 2, 4):
                _close(mx.mx_linear(x, w.tiled, n, elem=elem, cfg=a | b << 8 | nsl << 16), ref, bound)
        for m, cfg in ((5, 9), (5, 7 << 8), (5, 65 << 16), (150, 3), (150, 1 | 4 << 8), (150, 65 << 16)):
            with pytest.raises(L.BzError):
                mx.mx_linear(_rows(m, k, 23), w.tiled, n, elem=elem, cfg=cfg)


def test_threads_and_streams_at_once():
    """Products that slice K from host threads, on one stream and on their own."""
    import threading

    n, k = 1024, 8192
    w = Weight(n, k)
    xs = [_rows(m, k, 24 + m) for m in (5, 20, 40, 64)]
    want = [mx.mx_linear(x, w.tiled, n, elem="e4m3") for x in xs]
    torch.cuda.synchronize()
    for own_stream in (False, True):
        wrong = []

        def work(i):
            stream = torch.cuda.Stream() if own_stream else torch.cuda.current_stream()
            with torch.cuda.stream(stream):
                for _ in range(40):
                    got = mx.mx_linear(xs[i], w.tiled, n, elem="e4m3")
                    stream.synchronize()
                    if not torch.equal(got, want[i]):
                        wrong.append(i)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong


def test_two_graphs_at_once():
    """Two captured products that slice K, replayed on two streams."""
    n, k = 1024, 8192
    w = Weight(n, k)
    xs = [_rows(5, k, 30), _rows(48, k, 31)]
    want = [mx.mx_linear(x, w.tiled, n) for x in xs]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mx.mx_linear(x, w.tiled, n))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, want):
            assert torch.equal(o, e)
            o.zero_()
        torch.cuda.synchronize()


@pytest.mark.parametrize("rows", [3, 40])
def test_module_gradient_of_any_call(rows):
    lin = nn.Linear(256, 48, bias=False).cuda()
    mod, x = M4.Mxfp4Linear(lin), torch.randn(rows, 256, device="cuda", requires_grad=True)
    g = torch.randn(rows, 48, device="cuda").to(BF16)
    mod(x).backward(g.float())
    wq = O.rounded(_np(lin.weight), O.E2M1)
    ref = _np(g) @ wq
    _close(x.grad, ref, 2.0 ** -8 * np.abs(ref) + 48 * 2.0 ** -24 * (np.abs(_np(g)) @ np.abs(wq)))
    with torch.no_grad():
        assert torch.equal(mod(x), mod(x.detach()))


def test_large_row_offsets():
    """Rows whose codes and outputs lie past 2^31 bytes of one another."""
    m, k, n = 70_000, 16_384, 32
    x = torch.zeros(m, k, device="cuda", dtype=BF16)  # 2.3 GB
    tail = _rows(300, k, 32)
    x[-300:] = tail
    w = Weight(n, k)
    ref = mx.mx_linear(tail, w.tiled, n, elem="e4m3")
    out = mx.mx_linear(x, w.tiled, n, elem="e4m3")
    assert not out[:-300].any() and torch.equal(out[-300:], ref)
    codes, scales = mx.quantize_mx(x, "e4m3")
    assert torch.equal(mx.dequantize_mx(codes[-300:], scales[-300:], "e4m3"),
                       mx.dequantize_mx(*mx.quantize_mx(tail, "e4m3"), "e4m3"))
    del x, codes, scales
    wide = torch.empty(400, 6_000_000, device="cuda", dtype=BF16)  # rows 12 MB apart
    view = wide[:, 1024:1024 + k]
    view[:300] = tail
    assert torch.equal(mx.mx_linear(view[:300], w.tiled, n, elem="e4m3"), ref)
    few = mx.mx_linear(tail[:20], w.tiled, n, elem="e4m3")
    _close(mx.mx_linear(view[:20], w.tiled, n, elem="e4m3"), *_mx_reference(tail[:20], w, "e4m3", None, BF16))
    assert few.shape == (20, n)


def test_more_small_tiles_than_a_launch_holds():
    """The launch shapes with the smallest tiles are passed over, not the call refused."""
    m, n, k = 270_000, 131_072, 128
    x, w = _rows(400, k, 33), Weight(n, k)
    big = torch.zeros(m, k, device="cuda", dtype=BF16)
    big[:200], big[-200:] = x[:200], x[200:]
    out = mx.mx_linear(big, w.tiled, n)  # 71 GB
    few = mx.mx_linear(x, w.tiled, n)
    assert torch.equal(out[:200], few[:200]) and torch.equal(out[-200:], few[200:]) and not out[m // 2].any()
    del out, big
    torch.cuda.empty_cache()


def test_rows_that_are_not_of_their_shape():
    w, q = Weight(32, 256), mx.mx_rows(_rows(40, 256))
    for data, shape in ((q.data[:-16], q.shape), (q.data, (64, 256)), (q.data, (40, 128))):
        with pytest.raises(ValueError):
            mx.mx_linear(mx.MxRows(data, shape, q.elem), w.tiled, 32)
    with pytest.raises(ValueError, match="MxRows"):
        mx.mx_linear(mx.MxRows(q.data, q.shape, O.E4M3), w.tiled, 32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        mx.mx_linear(mx.MxRows(q.data.cpu(), q.shape, q.elem), w.tiled.cpu(), 32)


def test_calls_after_a_planned_one():
    """The second call of a shape is made by the binding: what differs from the first is seen, or refused."""
    n, k = 1024, 2048
    w, x = Weight(n, k), _rows(2, k, 40)
    res, gamma = _rows(2, n, 41), _rows(1, k, 42)[0]
    first = G.gemv(x, w.tiled, w.fmt, n)
    want = mx.mx_linear(x, w.tiled, n)
    for _ in range(3):
        assert torch.equal(G.gemv(x, w.tiled, w.fmt, n), first) and torch.equal(mx.mx_linear(x, w.tiled, n), want)
    for bad in (w.tiled[:-16], w.tiled.cpu()):
        for call in (lambda: G.gemv(x, bad, w.fmt, n), lambda: mx.mx_linear(x, bad, n)):
            with pytest.raises((ValueError, RuntimeError)):
                call()
    with pytest.raises(RuntimeError, match="no gradient"):
        mx.mx_linear(x.clone().requires_grad_(), w.tiled, n)
    with torch.no_grad():
        assert torch.equal(mx.mx_linear(x.clone().requires_grad_(), w.tiled, n), want)
    # rows to copy, to convert, of a wider tensor, of another type; types of the result and the residual
    wide = torch.empty(2, k + 8, device="cuda", dtype=BF16)
    wide[:, 8:] = x
    odd = torch.empty(2, k + 1, device="cuda", dtype=BF16)
    odd[:, 1:] = x
    for view in (wide[:, 8:], odd[:, 1:], x.float(), x.t().contiguous().t(), torch.nn.Parameter(x, requires_grad=False)):
        assert torch.equal(G.gemv(view, w.tiled, w.fmt, n), first) and torch.equal(mx.mx_linear(view, w.tiled, n), want)
        for elem in ELEMS:
            for a, b in zip(mx.quantize_mx(view, elem), mx.quantize_mx(x, elem)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for r in (res, res.float(), res.t().contiguous().t(), res[:1].expand(2, n)):
        for dt in (BF16, F32):
            a = G.gemv(x, w.tiled, w.fmt, n, epilogue=G.EPI_RESIDUAL, residual=r.contiguous(), out_dtype=dt)
            assert a.dtype == dt
            if r.stride(0) >= n:
                assert torch.equal(G.gemv(x, w.tiled, w.fmt, n, epilogue=G.EPI_RESIDUAL, residual=r, out_dtype=dt), a)
            b = mx.mx_linear(x, w.tiled, n, residual=r.contiguous(), out_dtype=dt)
            assert b.dtype == dt and torch.equal(mx.mx_linear(x, w.tiled, n, residual=r, out_dtype=dt), b)
    for bad in (res[:1], res[:, :-1], res.cpu()):
        for call in (lambda: G.gemv(x, w.tiled, w.fmt, n, epilogue=G.EPI_RESIDUAL, residual=bad),
                     lambda: mx.mx_linear(x, w.tiled, n, residual=bad)):
            with pytest.raises((ValueError, RuntimeError)):
                call()
    normed = G.gemv(x, w.tiled, w.fmt, n, gamma=gamma)
    assert torch.equal(G.gemv(x, w.tiled, w.fmt, n, gamma=gamma.float()), normed)
    with pytest.raises(ValueError):
        G.gemv(x, w.tiled, w.fmt, n, gamma=gamma[:-1])
    assert not torch.equal(G.gemv(x, w.tiled, w.fmt, n, gamma=gamma, eps=1), normed)


def test_a_plan_goes_with_the_table(monkeypatch):
    """A launch shape from a new table is taken, also for a shape that was called before."""
    from breeze_amd import tuning

    n, k = 1024, 2048
    w, x = Weight(n, k), _rows(1, k, 43)
    want = G.gemv(x, w.tiled, w.fmt, n)
    arch = tuning.arch_of(x.device)
    key = tuning.table_key(arch, n, k, w.fmt, G.EPI_NONE, False, 1)
    monkeypatch.setitem(tuning._TABLES, arch, {key: [0, 0, 0, 9]})  # (no such path)
    with pytest.raises(L.BzError):
        G.gemv(x, w.tiled, w.fmt, n)
    monkeypatch.setitem(tuning._TABLES, arch, {key: [0, 4, 0, 5]})
    _close(G.gemv(x, w.tiled, w.fmt, n), *_gemv_reference(x, w, G.EPI_NONE, None, 0.0, None, BF16))
    monkeypatch.undo()
    assert torch.equal(G.gemv(x, w.tiled, w.fmt, n), want)


def test_planned_calls_hold_no_memory():
    n, k = 1024, 8192
    w, x = Weight(n, k), _rows(5, k, 44)

    def calls():
        mx.mx_linear(x, w.tiled, n, elem="e4m3")  # (with a workspace)
        G.gemv(x, w.tiled, w.fmt, n)
        mx.dequantize_mx(*mx.quantize_mx(x))

    for _ in range(3):
        calls()
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    for _ in range(50):
        calls()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == held


@pytest.mark.parametrize("elem", ELEMS)
def test_few_rows_share_operands(elem):
    """Up to 8 rows leave room for their next units: every row on its own, whatever the others hold."""
    for n, k in ((48, 1664), (272, 640), (32, 1024)):
        w = Weight(n, k)
        for m in (1, 2, 3, 4, 5, 7, 8, 9):
            x = _rows(m, k, 50 + m)
            ref, bound = _mx_reference(x, w, elem, None, BF16)
            for t, upw, nsl in ((0, 0, 0), (1, 2, 1), (2, 3, 1), (1, 3, 2), (3, 4, 1), (1, 5, 3), (2, 6, 1), (1, 8, 2)):
                if upw * 8 < -(-k // 128) / max(nsl, 1):
                    continue  # (more units than 8 waves hold)
                cfg = t | upw << 8 | nsl << 16
                out = mx.mx_linear(x, w.tiled, n, elem=elem, cfg=cfg)
                _close(out, ref, bound)
                for r in range(m):
                    bad = x.clone()
                    bad[r, ::128 * 3] = float("nan")
                    got = mx.mx_linear(bad, w.tiled, n, elem=elem, cfg=cfg)
                    assert got[r].isnan().all() and torch.equal(got[:r], out[:r]) and torch.equal(got[r + 1:], out[r + 1:])


def test_a_refused_call_stays_refused():
    """What the library or the checks refuse is refused the second time too."""
    n, k = 64, 256
    x, m = _rows(2, k, 60), Weight(n, k)
    codes = torch.zeros(G.tiled_bytes(G.W_INT4_TILED, n, k), dtype=torch.uint8, device="cuda")
    for _ in range(3):
        G.gemv(x, codes, G.W_INT4_TILED, n)
        for kw in ({"group": 64}, {"epilogue": G.EPI_SILU_GATE}, {"epilogue": 7}):
            with pytest.raises((L.BzError, ValueError)):
                G.gemv(x, codes, G.W_INT4_TILED, n, **kw)
        for fmt in (G.W_MXFP4, 9, G.W_MXFP4_TILED_PAIRED):
            with pytest.raises((L.BzError, ValueError)):
                G.gemv(x, m.tiled, fmt, n)
        with pytest.raises((L.BzError, ValueError)):
            G.gemv(x, m.tiled, m.fmt, n - 8)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_prompts_after_a_planned_one(dtype):
    n, k, m = 256, 1024, 77
    w, x = Weight(n, k), _rows(m, k, 70, dtype)
    res = _rows(m, n, 71)
    wide = torch.empty(m, k + 3, device="cuda", dtype=dtype)
    wide[:, 3:] = x
    for elem in ELEMS:
        ref, bound = _mx_reference(x, w, elem, None, BF16)
        first = mx.mx_linear(x, w.tiled, n, elem=elem)
        _close(first, ref, bound)
        for view in (x, wide[:, 3:], x.t().contiguous().t()):
            for _ in range(2):
                assert torch.equal(mx.mx_linear(view, w.tiled, n, elem=elem), first)
        added = mx.mx_linear(x, w.tiled, n, elem=elem, residual=res, out_dtype=F32)
        _close(added, *_mx_reference(x, w, elem, res, F32))
        assert torch.equal(mx.mx_linear(x, w.tiled, n, elem=elem, residual=res.float(), out_dtype=F32), added)
        with pytest.raises(RuntimeError, match="no gradient"):
            mx.mx_linear(x.clone().requires_grad_(), w.tiled, n, elem=elem)
        with pytest.raises(ValueError):
            mx.mx_linear(x, w.tiled[:-16], n, elem=elem)
    xb = x.to(BF16)
    first = G.dequant_matmul(xb, w.tiled, w.fmt, n, k)
    _close(first, *_gemv_reference(xb, w, G.EPI_NONE, None, 0.0, None, BF16))
    for view in (xb, wide[:, 3:], wide.to(BF16)[:, 3:], x):
        assert torch.equal(G.dequant_matmul(view, w.tiled, w.fmt, n, k), first)
    for args in ((xb, w.tiled[:-16], w.fmt, n, k), (xb, w.tiled, w.fmt, n, k - 128), (xb, w.tiled, w.fmt, n - 8, k),
                 (xb, w.tiled, G.W_MXFP4_TILED_PAIRED, n, k)):
        for _ in range(2):
            with pytest.raises((ValueError, L.BzError)):
                G.dequant_matmul(*args)
    xg = xb.clone().requires_grad_()
    G.dequant_matmul(xg, w.tiled, w.fmt, n, k).sum().backward()
    assert xg.grad is not None
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(xb, torch.ones_like(xb))
        out = G.dequant_matmul(dual, w.tiled, w.fmt, n, k)
        assert torch.autograd.forward_ad.unpack_dual(out).tangent is not None
    assert G.dequant_matmul(xb[:0], w.tiled, w.fmt, n, k).shape == (0, n)


def test_launch_shapes_of_each_call():
    """Plans that a thread keeps: the last of each place, whatever was asked for between."""
    n, k = 256, 2048
    w = Weight(n, k)
    xs = {m: _rows(m, k, 80 + m) for m in range(33, 160, 9)}
    first = {m: (mx.mx_linear(x, w.tiled, n), mx.mx_linear(x, w.tiled, n, elem="e4m3"),
                 G.dequant_matmul(x, w.tiled, w.fmt, n, k)) for m, x in xs.items()}
    for m, x in reversed(xs.items()):
        ref, bound = _mx_reference(x, w, O.E2M1, None, BF16)
        _close(mx.mx_linear(x, w.tiled, n, cfg=1 | 2 << 8 | 2 << 16), ref, bound)
        again = (mx.mx_linear(x, w.tiled, n), mx.mx_linear(x, w.tiled, n, elem="e4m3"),
                 G.dequant_matmul(x, w.tiled, w.fmt, n, k))
        for a, b in zip(first[m], again):
            assert torch.equal(a, b)
