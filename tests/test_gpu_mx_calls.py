"""Calls of the microscaled operators at the edges of what they take, on the GPU."""

from __future__ import annotations

import pytest
import torch

from breeze_amd import gemv as G
from breeze_amd import tuning
from tests.test_gpu_mx import BF16, Weight, _close, _gemv_reference, _rows

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
