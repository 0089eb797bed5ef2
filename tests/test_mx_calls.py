"""Calls of the microscaled operators at the edges of what they take, without a GPU."""

from __future__ import annotations

import shutil
import subprocess
import threading
from pathlib import Path

import pytest
import torch

from breeze_amd import _lib as L
from breeze_amd import build as B
from breeze_amd import gemv as G
from breeze_amd import mx
from breeze_amd import mxfp4_linear as M4  # noqa: F401  (registers its operator)

CSRC = Path(__file__).resolve().parents[1] / "breeze-tts-2_amd" / "csrc"


# ---- rows cut into launches -------------------------------------------------------------------------


ROW_RUNS = """
#include <cstdio>
#include "bz_row_runs.h"
int main() {
    const int cases[][2] = {%s};
    for (auto& c : cases) {
        int64_t next = 0;
        int runs = 0;
        const int rc = bz::for_row_runs(c[0], c[1], [&](int64_t m0, int rows) {
            if (m0 != next || rows < 1 || (int64_t)rows * (c[1] / 8) > (int64_t)1 << 31) return 1;
            next = m0 + rows;
            return ++runs > 1000 ? 2 : 0;
        });
        std::printf("%%d %%lld %%d\\n", rc, (long long)next, runs);
    }
    return bz::for_row_runs(7, 32, [](int64_t, int) { return 5; }) == 5 ? 0 : 1;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_row_runs_cover_every_row_once(tmp_path):
    """Up to 2^31 - 1 rows: a first row past 2^31 was a write 34 GB before the buffer."""
    rows = [1, 2 ** 29, 2 ** 29 + 1, 3 * 2 ** 29, 3 * 2 ** 29 + 1, 2 ** 31 - 1]
    cases = [(m, 32) for m in rows] + [(2 ** 31 - 1, 64), (9, 2 ** 31 - 32), (2 ** 20, 2 ** 16)]
    (tmp_path / "runs.cpp").write_text(ROW_RUNS % ", ".join(f"{{{m}, {k}}}" for m, k in cases))
    exe = tmp_path / "runs"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}",
                    str(tmp_path / "runs.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    for (m, k), line in zip(cases, out):
        rc, end, runs = map(int, line.split())
        per = min(m, 2 ** 31 // (k // 8))
        assert rc == 0 and end == m and runs == -(-m // per), (m, k, line)


# ---- buffers of another device ------------------------------------------------------------------------


def test_scales_and_outputs_of_another_device_are_refused(monkeypatch):
    """A kernel would read or write their host addresses.  The meta device stands for the GPU."""
    def require(name, t, device):
        if t.device != device:
            raise RuntimeError(f"{name} is on {t.device}, expected {device}")

    def zeros(*shape, device="meta", dtype=torch.uint8):
        return torch.zeros(*shape, device=device, dtype=dtype)

    monkeypatch.setattr(G, "_require_gpu", require)
    w, sc, tiled = zeros(16, 64), zeros(16, 4), G.tiled_bytes(G.W_MXFP4_TILED, 16, 128)
    for name, call in (
            ("sc0", lambda: G.pack_tiled(G.W_MXFP4, w, 128, G.W_MXFP4_TILED, sc0=sc.new_zeros(16, 4, device="cpu"))),
            ("out", lambda: G.pack_tiled(G.W_MXFP4, w, 128, G.W_MXFP4_TILED, sc0=sc, out=zeros(tiled, device="cpu"))),
            ("out", lambda: G.pack_tiled(G.W_MXFP4_TILED, zeros(tiled), 128, G.W_MXFP4_TILED, n_total=32,
                                         out=zeros(2 * tiled, device="cpu"))),
            ("sc0", lambda: G.dequant(G.W_MXFP4, w, 16, 128, sc0=zeros(16, 4, device="cpu"))),
            ("sc1", lambda: G.dequant(G.W_INT4_MIN, w, 16, 128, sc0=zeros(16, dtype=torch.bfloat16),
                                      sc1=zeros(16, device="cpu", dtype=torch.bfloat16)))):
        with pytest.raises(RuntimeError, match=f"{name} is on cpu"):
            call()


# ---- sizes past 32 bits -------------------------------------------------------------------------------


def test_sizes_past_32_bits_are_refused(monkeypatch):
    """ctypes cuts an int to 32 bits: a row of 2^32 + 128 columns was taken for one of 128.  The meta device stands
    for the GPU."""
    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, device="meta", dtype=dtype)

    launched = []
    monkeypatch.setattr(mx, "_gpu", lambda *a: None)
    monkeypatch.setattr(mx, "_call", lambda *a: launched.append(a))
    u8 = torch.uint8
    w = meta(1280, dtype=u8)
    for m, k in ((1, 2 ** 32 + 128), (1, 2 ** 31), (2 ** 32 + 1, 128)):
        for call in (lambda: mx.quantize_mx(meta(m, k)), lambda: mx.mx_rows(meta(m, k)),
                     lambda: mx.mx_linear(meta(m, k), w, 16),
                     lambda: mx.dequantize_mx(meta(m, k // 2, dtype=u8), meta(m, k // 32, dtype=u8))):
            with pytest.raises(ValueError, match="2\\^31"):
                call()
    for n in (2 ** 32 + 16, 16 - 2 ** 32):
        with pytest.raises(ValueError, match="W_MXFP4_TILED"):
            mx.mx_linear(meta(1, 128), w, n)
        for fmt, size in ((G.W_MXFP4_TILED, 1280), (G.W_INT4_TILED, 1152), (G.W_FP8_TILED, 2176)):
            assert G.tiled_bytes(fmt, 16, 128) == size and G.tiled_bytes(fmt, n, 128) == G.tiled_bytes(fmt, 16, n) == 0
            with pytest.raises(ValueError, match="cannot be tiled"):
                G._check_weight(torch.zeros(size, dtype=u8), fmt, n, 128, 128, None, None)
    assert not launched


# ---- workspaces of host threads -------------------------------------------------------------------------


@pytest.mark.parametrize("held", [False, True])
def test_threads_that_need_a_workspace_at_once(monkeypatch, held):
    """No buffer that a thread was given is dropped while the other allocates: the thread is about to launch on it."""
    zeros, inside = torch.zeros, threading.Barrier(2)

    def slow(*args, **kw):  # the other thread gets as far as its own allocation, where nothing keeps it from that
        try:
            inside.wait(0.5)
        except threading.BrokenBarrierError:
            pass
        return zeros(*args, **kw)

    table, retired, given = {}, [], []
    monkeypatch.setattr(L, "capture_of", lambda stream: None)
    args = (torch.device("cpu"), 7, retired)
    if held:
        given.append(L.stream_workspace(table, ("key",), 100, *args).data_ptr())
    monkeypatch.setattr(torch, "zeros", slow)

    def work(nbytes):
        buf = L.stream_workspace(table, ("key",), nbytes, *args)
        assert buf.numel() * 4 >= nbytes
        given.append(buf.data_ptr())

    threads = [threading.Thread(target=work, args=(n,)) for n in (3 << 20, (3 << 20) + 4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    kept = {b.data_ptr() for b in [*table.values(), *retired]}
    assert len(table) == 1 and len(given) == 2 + held and set(given) <= kept


def test_a_workspace_asked_for_inside_an_allocation(monkeypatch):
    """A finaliser that runs in the allocation and asks for the same workspace: its buffer stays alive too."""
    zeros, table, retired, given = torch.zeros, {}, [], []
    monkeypatch.setattr(L, "capture_of", lambda stream: None)

    def nested(*args, **kw):
        monkeypatch.setattr(torch, "zeros", zeros)
        given.append(L.stream_workspace(table, ("key",), 100, torch.device("cpu"), 7, retired).data_ptr())
        return zeros(*args, **kw)

    monkeypatch.setattr(torch, "zeros", nested)
    given.append(L.stream_workspace(table, ("key",), 2 << 20, torch.device("cpu"), 7, retired).data_ptr())
    assert [b.data_ptr() for b in retired] + [table["key", 7, None].data_ptr()] == given


# ---- what autograd follows ------------------------------------------------------------------------------


def test_what_autograd_follows():
    x = torch.ones(2, 64)
    assert not mx.followed(x)
    p = x.clone().requires_grad_()
    assert mx.followed(p) and mx.followed(2 * p) and not mx.followed(p.detach())
    with torch.no_grad():
        assert not mx.followed(p)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        assert mx.followed(dual) and mx.followed(2 * dual) and not mx.followed(x)
        with torch.no_grad():
            assert mx.followed(dual)  # (no_grad is about the backward pass)
        for f in (mx.quantize_mx, mx.mx_rows):
            with pytest.raises(RuntimeError, match="no gradient|GPU tensor"):
                f(dual)


# ---- traced calls ---------------------------------------------------------------------------------------


def test_the_traced_modules_operator_has_a_shape():
    x = torch.empty(77, 256, device="meta", dtype=torch.bfloat16)
    out = torch.ops.breeze_amd.mxfp4_linear(x, torch.empty(3, 2304, device="meta", dtype=torch.uint8), 48, 8)
    assert out.shape == (77, 48) and out.dtype == torch.bfloat16


# ---- few rows in one launch -------------------------------------------------------------------------------


@pytest.mark.parametrize("elem", [L.MX_E2M1, L.MX_E4M3])
def test_the_built_in_shape_of_few_rows_fits(elem):
    """17 .. 32 rows: the rule's shape did not fit LDS at about one in eight sizes, and the call was refused."""
    need = L.lib().bz_mx_gemv_workspace
    for m in (1, 5, 8, 9, 16, 17, 25, 32):
        for n, k in ((4096, 10240), (3584, 10240), (8192, 5120), (14336, 4096), (20480, 4096), (32768, 2560),
                     (151936, 2560), (576, 65536)):
            assert need(elem, m, n, k, 0) < 1 << 31, (m, n, k)
        for n in [*range(16, 20481, 1040), 32768]:
            for k in range(128, 10241, 640):
                assert need(elem, m, n, k, 0) < 1 << 31, (m, n, k)
        assert need(elem, m, 64, (1 << 22) + 128, 0) == (1 << 64) - 1
    for cfg in (8 | 1 << 8 | 1 << 16, 8 | 2 << 8 | 1 << 16):  # 16 waves over eight blocks of 32 rows: 256 KiB of sums
        assert need(elem, 32, 512, 2048 * (cfg >> 8 & 255), cfg) == (1 << 64) - 1
    assert need(elem, 32, 512, 2048, 8 | 1 << 16) == 0  # (the rule's units, more of them)


# ---- views that share memory ------------------------------------------------------------------------------


def test_views_overlap_where_they_share_an_element():
    buf = torch.zeros(6, 20)
    marks = torch.arange(120).view(6, 20)
    views = [lambda t: t[:, :8], lambda t: t[:, 8:], lambda t: t[:, 7:12], lambda t: t[:, 12:], lambda t: t[1:4, 2:9],
             lambda t: t[4:, :8], lambda t: t[:1, 3:15], lambda t: t.view(-1)[15:115].view(5, 20)[:, :8],
             lambda t: t.view(-1)[15:115].view(5, 20)[:, 9:], lambda t: t[:, 2:9:2], lambda t: t.t()[:, 1:3],
             lambda t: t[::2, :8], lambda t: t[1::2, :8], lambda t: t.view(-1), lambda t: t[2:2]]
    for f in views:
        for g in views:
            share = bool(set(f(marks).flatten().tolist()) & set(g(marks).flatten().tolist()))
            said = mx._overlap(f(buf), g(buf))
            rows = all(v.dim() == 2 and v.stride(1) == 1 and v.stride(0) == 20 for v in (f(buf), g(buf)))
            assert said >= share and (not rows or said == share), (f(marks), g(marks))
    half = torch.zeros(6, 40, dtype=torch.bfloat16)
    assert not mx._overlap(half[:, :32], half.view(torch.float32)[:, 16:])
    assert mx._overlap(half[:, :33], half.view(torch.float32)[:, 16:])


# ---- the build's scratch guard ------------------------------------------------------------------------------


def test_the_scratch_guard_names_each_kernel():
    """One pattern a kernel: an alternative of several would pass while any one of them is compiled."""
    assert not [p for p in B.NO_SCRATCH + B.NO_SCRATCH_MX if "|" in p]
    kernels = [(f"_ZN2bz{len(p)}{p}ILi0EEEv", 64, 0) for p in B.NO_SCRATCH_MX]
    assert {p for p in B.NO_SCRATCH_MX} == {"mx_gemm", "mx_gemv", "mx_quantize_rows", "mx_quantize_tiled", "mx_dequantize_rows"}
    B.check_scratch(kernels, B.NO_SCRATCH_MX)
    for i, (name, vgpr, _) in enumerate(kernels):
        with pytest.raises(RuntimeError, match="no compiled kernel"):
            B.check_scratch(kernels[:i] + kernels[i + 1:], B.NO_SCRATCH_MX)
        with pytest.raises(RuntimeError, match="scratch"):
            B.check_scratch(kernels[:i] + [(name, vgpr, 16)] + kernels[i + 1:], B.NO_SCRATCH_MX)
    built = B.PKG_DIR / "_build" / "kernel_resources.txt"
    if built.exists():  # (the names of the last build)
        names = [(line.split()[-1], 0, 0) for line in built.read_text().splitlines()]
        B.check_scratch(names, B.NO_SCRATCH + B.NO_SCRATCH_MX)
