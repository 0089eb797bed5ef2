"""Calls of the microscaled operators at the edges of what they take, on the GPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from torch import nn

from oracle import bz_mx_oracle as O

from breeze_amd import _lib as L
from breeze_amd import gemv as G
from breeze_amd import mx
from breeze_amd import mxfp4_linear as M4
from breeze_amd import tuning
from tests.test_gpu_mx import BF16, ELEMS, Weight, _close, _gemv_reference, _mx_reference, _np, _rows

pytestmark = pytest.mark.gpu


def test_a_table_replaced_while_the_workspace_is_made(monkeypatch):
    """The binding holds nothing of the launch-shape table while it runs Python."""
    m, n, k = 13, 1024, 8192
    w, x = Weight(n, k), _rows(m, k, 1)
    want = G.gemv(x, w.tiled, w.fmt, n)
    _close(want, *_gemv_reference(x, w, G.EPI_NONE, None, 0.0, None, BF16))
    arch = tuning.arch_of(x.device)
    key = ("tiled", w.fmt, n, k, G.EPI_NONE, False, m)
    assert tuning._table(arch)[key][3] > 0  # this shape asks for a workspace
    raw, calls, other = G._raw_workspace, [], []

    def replacing(*args):
        calls.append(args)
        tuning._TABLES[arch].clear()
        tuning._TABLES[arch] = {}
        other.extend((i, -i, i * i, 9, 9) for i in range(2000))  # (tuples where the plan's were)
        return raw(*args)

    n_out, size, cfg, need = tuning._table(arch)[key]
    monkeypatch.setitem(tuning._TABLES, arch, {key: (n_out, size, tuple(list(cfg)), need)})  # (nothing else holds it)
    monkeypatch.setattr(G, "_raw_workspace", replacing)
    assert torch.equal(G.gemv(x, w.tiled, w.fmt, n), want) and len(calls) == 1
    monkeypatch.undo()
    assert torch.equal(G.gemv(x, w.tiled, w.fmt, n), want)


# ---- what autograd follows ------------------------------------------------------------------------------


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("m", [2, 40])
def test_what_autograd_follows_is_refused(elem, m):
    """Rows, residuals and outputs, followed backward or forward, the first time and after a planned call."""
    n, k = 64, 256
    w, x, res = Weight(n, k), _rows(m, k, 2), _rows(m, n, 3)
    want, codes = mx.mx_linear(x, w.tiled, n, elem=elem, residual=res), mx.quantize_mx(x, elem)[0]
    for _ in range(2):
        p, r, o = x.clone().requires_grad_(), res.clone().requires_grad_(), res.clone().requires_grad_()
        calls = [lambda: mx.quantize_mx(p, elem), lambda: mx.mx_rows(p, elem), lambda: mx.mx_linear(p, w.tiled, n, elem=elem),
                 lambda: mx.mx_linear(x, w.tiled, n, elem=elem, residual=r),
                 lambda: mx.mx_linear(mx.mx_rows(x, elem), w.tiled, n, residual=r),
                 lambda: mx.mx_linear(x, w.tiled, n, elem=elem, residual=res, out=o)]
        for call in calls:
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
        with torch.no_grad():
            for call in calls:
                call()
            assert torch.equal(mx.mx_linear(p, w.tiled, n, elem=elem, residual=r), want) and torch.equal(o, want)
        assert torch.equal(mx.quantize_mx(p.detach(), elem)[0].view(torch.uint8), codes.view(torch.uint8))
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual
            p, r = dual(x, torch.ones_like(x)), dual(res, torch.ones_like(res))
            for call in calls[:-1]:
                with pytest.raises(RuntimeError, match="no gradient"):
                    call()
            assert torch.equal(mx.mx_linear(x, w.tiled, n, elem=elem, residual=res), want)


def test_a_parameter_is_quantized_as_it_is():
    p = torch.nn.Parameter(_rows(48, 256, 4))
    assert torch.equal(M4.quantize_mxfp4(p), M4.quantize_mxfp4(p.data))


@pytest.mark.parametrize("rows", [1, 3, 32, 40])
@pytest.mark.parametrize("n,k", [(48, 256), (50, 200)])
def test_module_keeps_forward_tangents(rows, n, k):
    lin = nn.Linear(k, n, bias=False).cuda()
    x, t = torch.randn(rows, k, device="cuda"), torch.randn(rows, k, device="cuda").to(BF16)
    wq = O.rounded(np.pad(_np(lin.weight), ((0, 0), (0, -k % 32))), O.E2M1)[:, :k]
    ref = _np(t) @ wq.T
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, t.float())
        out = M4.Mxfp4Linear(lin)(dual)
        value, tangent = torch.autograd.forward_ad.unpack_dual(out)
        # the tangent of a bf16 product, rounded once to bf16
        _close(tangent, ref, 2.0 ** -8 * np.abs(ref) + k * 2.0 ** -24 * (np.abs(_np(t)) @ np.abs(wq).T))
        for bits in (4, 8):
            mod = M4.Mxfp4Linear(lin, act_bits=bits)
            with pytest.raises(RuntimeError, match="no gradient"):
                mod(dual)
            assert mod(x).shape == (rows, n)


@pytest.mark.parametrize("act_bits", [16, 8, 4])
@pytest.mark.parametrize("n,k", [(64, 256), (50, 200)])
def test_a_compiled_module_multiplies_what_an_eager_one_does(act_bits, n, k):
    """Row counts on either side of a prompt's, one compilation for all of them."""
    mod = M4.Mxfp4Linear(nn.Linear(k, n, bias=False).cuda(), act_bits=act_bits)
    torch._dynamo.reset()
    compiled = torch.compile(mod, fullgraph=True, backend="eager", dynamic=True)
    with torch.no_grad():
        for rows in (5, 32, 33, 70, 200, 2):
            x = _rows(rows, k, rows)
            assert torch.equal(compiled(x), mod(x)), rows
        x = _rows(60, k, 7).view(3, 20, k)
        assert torch.equal(compiled(x), mod(x))
    torch._dynamo.reset()


def test_the_traced_modules_operator():
    mod = M4.Mxfp4Linear(nn.Linear(256, 48, bias=False).cuda(), act_bits=8)
    for rows in (4, 40):
        torch.library.opcheck(M4.mxfp4_linear_op, (_rows(rows, 256, 5), mod.weight_mxfp4, 48, 8),
                              test_utils=("test_schema", "test_faketensor"))


# ---- plans that calls leave behind --------------------------------------------------------------------


def test_plans_are_few_and_of_calls_that_were_made(monkeypatch):
    n, k = 64, 256
    w = Weight(n, k)
    monkeypatch.setattr(mx, "_PLANS", {})
    for m in (2, 40):
        x = _rows(m, k, m)
        for kw in ({"residual": x}, {"out_dtype": torch.float16}, {"out": x[:, :n]}, {"cfg": 1 | 2 << 8}):
            try:
                mx.mx_linear(x, w.tiled, n, **kw)
            except (ValueError, TypeError):
                pass
        with pytest.raises(ValueError):
            mx.mx_linear(x, w.tiled[:-16], n)
        assert mx.mx_linear(x[:0], w.tiled, n).shape == (0, n)
    assert not mx._PLANS
    monkeypatch.setattr(mx, "_MOST_PLANS", 20)
    base = _rows(150, k, 9)
    want = mx.mx_linear(base, w.tiled, n)
    for _ in range(2):
        for m in range(1, 151):
            out = mx.mx_linear(base[:m], w.tiled, n)
            assert len(mx._PLANS) <= 20 and torch.equal(mx.mx_linear(base[:m], w.tiled, n), out)
    assert torch.equal(out, want)


# ---- few rows in one launch -------------------------------------------------------------------------------


@pytest.mark.parametrize("n,k", [(4096, 10240), (8192, 5120), (14336, 4096), (20480, 4096), (32768, 2560), (32784, 128),
                                 (2624, 16384)])
def test_few_rows_whose_sums_would_not_fit(n, k):
    w = Weight(n, k)
    for m in (17, 32):
        x, res = _rows(m, k, m), _rows(m, n, 6)
        for elem in ELEMS:
            ref, bound = _mx_reference(x, w, elem, res, BF16)
            for cfg in (0, 4, 3 << 16):
                if elem == O.E4M3 and k == 16384 and cfg == 3 << 16:  # 8 waves hold 40 units, a slice has 43
                    with pytest.raises(L.BzError):
                        mx.mx_linear(x, w.tiled, n, elem=elem, residual=res, cfg=cfg)
                    continue
                out = mx.mx_linear(x, w.tiled, n, elem=elem, residual=res, cfg=cfg)
                _close(out, ref, bound)
                assert torch.equal(mx.mx_linear(x, w.tiled, n, elem=elem, residual=res, cfg=cfg), out)
            assert mx._PLANS[mx._ELEM[elem], m, n, k][1] == (n <= mx.ONE_ROUND)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("m", [1, 3, 40])
def test_rows_residual_and_output_in_one_buffer(elem, m):
    """Column ranges of one tensor that share no element."""
    n, k = 144, 256
    w = Weight(n, k)
    buf = torch.randn(m, n + k + n + 8).to(BF16).cuda()
    out, x, res = buf[:, :n], buf[:, n:n + k], buf[:, n + k:n + k + n]
    before = buf.clone()
    ref, bound = _mx_reference(x, w, elem, res, BF16)
    mx.mx_linear(x, w.tiled, n, elem=elem, residual=res, out=out)
    _close(out, ref, bound)
    before[:, :n] = out
    assert torch.equal(buf, before)
    for wrong in (buf[:, 1:n + 1], buf[:, n + k - 1:n + k - 1 + n]):
        with pytest.raises(ValueError, match="overlap"):
            mx.mx_linear(x, w.tiled, n, elem=elem, out=wrong)


# ---- scale codes at the ends, rows with infinities ----------------------------------------------------------


def _product(x, w):
    """bf16 rows times the weight, by the call of their number."""
    if x.shape[0] <= 32:
        return G.gemv(x, w.tiled, w.fmt, w.n, out_dtype=torch.float32)
    return G.dequant_matmul(x, w.tiled, w.fmt, w.n, w.k)


def _scaled(n, k, codes):
    """A weight whose blocks take these scale codes in turn along a row."""
    w = Weight(n, k)
    w.scales[:] = np.resize(np.asarray(codes, np.uint8), w.scales.shape)
    w.tiled = torch.from_numpy(O.tile(w.codes, w.scales, O.E2M1)).cuda()
    w.values = O.values(w.codes, w.scales, O.E2M1)
    return w


MS = [1, 2, 5, 9, 17, 40]


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("n,k", [(48, 640), (272, 1280), (4112, 512)])
def test_products_of_the_smallest_scales(m, n, k):
    """Codes 0, 1 and 2: weights from 2^-128 up, some of them subnormal bf16, times rows about 2^100."""
    w = _scaled(n, k, [0, 1, 0, 2])
    x = (_rows(m, k, 8).float() * 2.0 ** 100).to(BF16)
    out_dtype = torch.float32 if m <= 32 else BF16
    _close(_product(x, w), *_gemv_reference(x, w, G.EPI_NONE, None, 0.0, None, out_dtype))
    for elem in ELEMS:
        _close(mx.mx_linear(x, w.tiled, n, elem=elem, out_dtype=torch.float32), *_mx_reference(x, w, elem, None, torch.float32))


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("n,k", [(48, 640), (272, 1280)])
def test_products_of_the_largest_scales(m, n, k):
    """Codes 252 to 254 times rows about 2^-110.  bf16 holds a weight below 2^128; a larger one is an infinity to the
    products of bf16 rows, and itself to those of quantised rows, whose scales the matrix cores add."""
    w = _scaled(n, k, [252, 254, 253, 254])
    x = (_rows(m, k, 9).float().abs() * 2.0 ** -110 + 2.0 ** -112).to(BF16)
    for elem in ELEMS:
        _close(mx.mx_linear(x, w.tiled, n, elem=elem, out_dtype=torch.float32), *_mx_reference(x, w, elem, None, torch.float32))
    got = _np(_product(x, w))
    with np.errstate(invalid="ignore"):
        want = _np(x) @ np.where(np.abs(w.values) < 2.0 ** 128, w.values, np.copysign(np.inf, w.values)).T
    assert (np.isnan(got) == np.isnan(want)).all() and (got[np.isinf(want)] == want[np.isinf(want)]).all()
    w.codes[:] = w.codes & 0xB  # elements up to 1.5
    w.tiled = torch.from_numpy(O.tile(w.codes, w.scales, O.E2M1)).cuda()
    w.values = O.values(w.codes, w.scales, O.E2M1)
    _close(_product(x, w), *_gemv_reference(x, w, G.EPI_NONE, None, 0.0, None, torch.float32 if m <= 32 else BF16))


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("n,k", [(48, 640), (272, 1280), (4112, 512)])
def test_products_of_blocks_that_are_nan(m, n, k):
    """Code 255: the columns of the result whose weight row has such a block, and no others."""
    w, x = Weight(n, k), _rows(m, k, 10)
    clean = [_product(x, w)] + [mx.mx_linear(x, w.tiled, n, elem=e) for e in ELEMS]
    bad = np.zeros(n, bool)
    for row, block in ((0, 0), (5, k // 32 - 1), (n - 1, 7), (n // 2, 3)):
        w.scales[row, block] = 255
        bad[row] = True
    w.tiled = torch.from_numpy(O.tile(w.codes, w.scales, O.E2M1)).cuda()
    bad = torch.from_numpy(bad).cuda()
    for out, was in zip([_product(x, w)] + [mx.mx_linear(x, w.tiled, n, elem=e) for e in ELEMS], clean):
        assert out[:, bad].isnan().all() and torch.equal(out[:, ~bad], was[:, ~bad])


@pytest.mark.parametrize("m", MS)
@pytest.mark.parametrize("n,k", [(48, 640), (272, 1280), (4112, 512), (64, 8192)])
def test_bf16_rows_with_nan_and_infinity(m, n, k):
    """An infinity times a weight of zero is a NaN, times another one of that one's sign; rows are independent."""
    w, x = Weight(n, k), _rows(m, k, 11)
    clean = _product(x, w)
    for r in sorted({0, m // 2, m - 1}):
        for bad in (float("inf"), -float("inf"), float("nan")):
            for col in (0, k // 2 + 3, k - 1):
                y = x.clone()
                y[r, col] = bad
                out = _product(y, w)
                assert torch.equal(out[:r], clean[:r]) and torch.equal(out[r + 1:], clean[r + 1:])
                weight = torch.from_numpy(w.values[:, col]).cuda()
                want = bad * weight
                assert torch.equal(out[r].isnan(), want.isnan()) and (out[r][~want.isnan()] == want[~want.isnan()]).all()


@pytest.mark.parametrize("m", [1, 2, 5, 9])
@pytest.mark.parametrize("epi", [G.EPI_NONE, G.EPI_SILU_GATE])
def test_normed_rows_with_nan_and_infinity(m, epi):
    n, k = 272, 640
    w, x, gamma = Weight(n, k, paired=epi == G.EPI_SILU_GATE), _rows(m, k, 12), _rows(1, k, 13)[0].abs() + 1

    def run(x):
        return G.gemv(x, w.tiled, w.fmt, n, gamma=gamma, epilogue=epi)

    clean = run(x)
    for r in sorted({0, m - 1}):
        for bad in (float("inf"), float("nan")):
            y = x.clone()
            y[r, 100] = bad
            out = run(y)
            assert out[r].isnan().all() and torch.equal(out[:r], clean[:r]) and torch.equal(out[r + 1:], clean[r + 1:])


@pytest.mark.parametrize("m", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("n,k", [(48, 640), (272, 1280), (64, 2176), (4112, 192), (64, 4160), (2560, 1280)])
def test_fp8_rows_with_infinity_in_the_last_unit(m, n, k):
    """The waves' units past a row multiply their zero weights by zeros, not by its last columns."""
    codes, scale = G.quantize_fp8_device(_rows(n, k, 14), 1e-12)
    w = G.pack_tiled(G.W_FP8, codes.view(torch.uint8), k, G.W_FP8_TILED, sc0=scale)
    values, x = G.dequant(G.W_FP8_TILED, w, n, k), _rows(m, k, 15)
    clean = G.gemv(x, w, G.W_FP8_TILED, n)
    for bad in (float("inf"), -float("inf")):
        y = x.clone()
        y[m - 1, k - 1] = bad
        out = G.gemv(y, w, G.W_FP8_TILED, n)
        want = bad * values[:, k - 1]
        assert torch.equal(out[:m - 1], clean[:m - 1]) and torch.equal(out[m - 1].isnan(), want.isnan())
        assert (out[m - 1][~want.isnan()] == want[~want.isnan()]).all()
