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
