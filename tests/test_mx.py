"""Operators over microscaled blocks without a GPU: refusals, sizes and the
oracle's own properties."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np
import pytest
import torch
from torch import nn

from oracle import bz_mx_oracle as O

from breeze_amd import _lib as L
from breeze_amd import gemv as G
from breeze_amd import mx
from breeze_amd import mxfp4_linear as M4
from breeze_amd import quantized_checkpoint as Q
from breeze_amd.fused import kernels as FK

HEADER = Path(__file__).resolve().parents[1] / "include" / "bz_mx.h"
FAKE = 1 << 20  # never dereferenced: the calls below fail validation


def test_enums_match_the_header():
    text = HEADER.read_text()
    pairs = re.findall(r"\bBZ_(MX_[A-Z0-9]+)\s*=\s*(\d+)", text) + re.findall(r"#define BZ_(MX_F16) (\d+)", text)
    assert {n for n, _ in pairs} >= {"MX_E2M1", "MX_E4M3", "MX_ROWS", "MX_TILED", "MX_F16"}
    for name, value in pairs:
        assert getattr(L, name) == int(value), name


def test_every_function_of_the_header_is_exported():
    names = set(re.findall(r"\b(bz_mx_[a-z]+(?:_[a-z]+)*)\(", HEADER.read_text()))
    assert names and names <= set(L.EXPORTS)


# ---- the oracle -----------------------------------------------------------------------------------


def test_oracle_e4m3_is_torchs_rounding():
    """Values whose block scale is 1: the elements are the type's own rounding."""
    rng = np.random.default_rng(0)
    x = rng.uniform(-448, 448, (64, 32)) * 2.0 ** rng.integers(-17, 1, (64, 32))
    x[:, 0] = 256 + 191 * rng.random(64)
    x = x.astype(np.float32)
    codes, scales = O.quantize(x.astype(np.float64), O.E4M3)
    assert (scales == 127).all()
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert (codes == want).all()


def test_oracle_e2m1_ties_go_to_the_even_code():
    x = np.zeros((1, 32))
    x[0, :16] = [4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 5.01, 7.9, -0.25, -0.75, -5, 0.2500001, 0.2499999, -0.0]
    codes, scales = O.quantize(x, O.E2M1)
    assert scales[0, 0] == 127
    got = O.values(codes, scales, O.E2M1)[0, :16]
    assert got.tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 6, 0, -1, -4, 0.5, 0, 0]


@pytest.mark.parametrize("elem", [O.E2M1, O.E4M3])
def test_oracle_rounds_by_at_most_half_a_step(elem):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 128)) * np.exp(rng.standard_normal((50, 1)) * 8)
    v = O.rounded(x, elem)
    a = np.abs(x.reshape(50, 4, 32)).max(-1, keepdims=True).repeat(32, -1).reshape(x.shape)
    s = 2.0 ** (np.floor(np.log2(a)) - O.EMAX[elem])
    rel, small, top = (2.0 ** -2, 0.25, 6) if elem == O.E2M1 else (2.0 ** -4, 2.0 ** -10, 448)
    inside = np.abs(x) <= top * s
    assert (np.abs(v - x)[inside] <= np.maximum(rel * np.abs(x), small * s)[inside]).all()
    assert (np.abs(v)[~inside] == (top * s)[~inside]).all()


# ---- sizes and refusals of the C ABI -----------------------------------------------------------------


def test_sizes():
    lib = L.lib()
    assert lib.bz_tiled_bytes(L.W_MXFP4_TILED, 16, 128) == 1024 + 256
    assert lib.bz_tiled_bytes(L.W_MXFP4_TILED_PAIRED, 32, 640) == 2 * (5 * 1024 + 512)
    assert lib.bz_tiled_bytes(L.W_MXFP4_TILED, 24, 128) == 0 and lib.bz_tiled_bytes(L.W_MXFP4_TILED, 16, 96) == 0
    assert lib.bz_tiled_bytes(L.W_MXFP4, 16, 128) == 0
    assert lib.bz_mx_rows_bytes(0, 17, 512) == 2 * (4 * 1024 + 256)
    assert lib.bz_mx_rows_bytes(1, 16, 512) == 4 * 2048 + 256
    for bad in ((2, 16, 128), (0, 0, 128), (0, 16, 96), (-1, 16, 128)):
        assert lib.bz_mx_rows_bytes(*bad) == 0
    codes = np.zeros((32, 640), np.uint8)
    assert O.tile(codes, codes[:, :20], O.E2M1).size == lib.bz_tiled_bytes(L.W_MXFP4_TILED, 32, 640)
    assert O.tile(codes[:17], codes[:17, :20], O.E4M3).size == lib.bz_mx_rows_bytes(1, 17, 640)


@pytest.mark.parametrize("kw,status", [
    ({"x": None}, L.ERR_INVALID_ARG), ({"codes": None}, L.ERR_INVALID_ARG), ({"M": 0}, L.ERR_INVALID_ARG),
    ({"K": 0}, L.ERR_INVALID_ARG), ({"ldx": 63}, L.ERR_INVALID_ARG), ({"elem": 2}, L.ERR_INVALID_ARG),
    ({"dt": 3}, L.ERR_INVALID_ARG), ({"layout": 2}, L.ERR_INVALID_ARG), ({"scales": None}, L.ERR_INVALID_ARG),
    ({"layout": 1, "K": 128, "ldx": 128}, L.ERR_INVALID_ARG),              # tiled rows carry their scales
    ({"K": 48, "ldx": 64}, L.ERR_SHAPE), ({"layout": 1, "scales": None}, L.ERR_SHAPE),
    ({"x": FAKE + 1}, L.ERR_ALIGNMENT), ({"dt": 1, "x": FAKE + 2}, L.ERR_ALIGNMENT), ({"codes": FAKE + 2}, L.ERR_ALIGNMENT),
    ({"layout": 1, "K": 128, "ldx": 128, "scales": None, "codes": FAKE + 8}, L.ERR_ALIGNMENT),
])
def test_quantize_arguments(kw, status):
    d = dict(x=FAKE, dt=0, ldx=64, M=3, K=64, elem=0, layout=0, codes=FAKE, scales=FAKE) | kw
    assert L.lib().bz_mx_quantize(d["x"], d["dt"], d["ldx"], d["M"], d["K"], d["elem"], d["layout"], d["codes"],
                                  d["scales"], None) == status


@pytest.mark.parametrize("kw,status", [
    ({"codes": None}, L.ERR_INVALID_ARG), ({"scales": None}, L.ERR_INVALID_ARG), ({"out": None}, L.ERR_INVALID_ARG),
    ({"M": -1}, L.ERR_INVALID_ARG), ({"ldo": 60}, L.ERR_INVALID_ARG), ({"elem": 5}, L.ERR_INVALID_ARG),
    ({"dt": 2}, L.ERR_INVALID_ARG), ({"K": 40, "ldo": 64}, L.ERR_SHAPE), ({"codes": FAKE + 1}, L.ERR_ALIGNMENT),
    ({"out": FAKE + 1}, L.ERR_ALIGNMENT), ({"dt": 1, "out": FAKE + 2}, L.ERR_ALIGNMENT),
])
def test_dequantize_arguments(kw, status):
    d = dict(codes=FAKE, scales=FAKE, elem=0, M=3, K=64, out=FAKE, dt=0, ldo=64) | kw
    assert L.lib().bz_mx_dequantize(d["codes"], d["scales"], d["elem"], d["M"], d["K"], d["out"], d["dt"], d["ldo"],
                                    None) == status


@pytest.mark.parametrize("kw,status", [
    ({"fmt": L.W_MXFP4}, L.ERR_INVALID_ARG),                               # a source format: no product reads it
    ({"fmt": L.W_MXFP4_TILED_PAIRED + 1}, L.ERR_INVALID_ARG),
    ({"epi": L.EPI_SILU_GATE}, L.ERR_UNSUPPORTED),                         # plain tiled + SiLU-gate
    ({"fmt": L.W_MXFP4_TILED_PAIRED}, L.ERR_UNSUPPORTED),                  # paired needs SiLU-gate
    ({"path": 4}, L.ERR_UNSUPPORTED), ({"path": 2}, L.ERR_UNSUPPORTED),    # paths 5 and 6 only
    ({"N": 72}, L.ERR_SHAPE), ({"K": 192}, L.ERR_SHAPE),
])
def test_gemv_arguments(kw, status):
    d = dict(fmt=L.W_MXFP4_TILED, N=64, K=256, epi=0, path=0) | kw
    desc = L.gemv_desc(L.ABI_VERSION, 1, d["N"], d["K"], 128, d["fmt"], d["epi"], 0, 0, 0, 0, 0, d["path"], 0, 1e-6,
                       FAKE, 256, FAKE, 0, 0, 0, 0, 0, FAKE, 128, 0, 0, 0, 0, 0, 0)
    assert L.lib().bz_gemv(desc, None) == status


@pytest.mark.parametrize("kw,status", [
    ({"src": L.W_INT4_ZP}, L.ERR_INVALID_ARG), ({"dst": L.W_INT4_TILED}, L.ERR_INVALID_ARG),
    ({"src": L.W_MXFP4_TILED_PAIRED}, L.ERR_INVALID_ARG), ({"sc": None}, L.ERR_INVALID_ARG),
    ({"row0": 8, "N": 16}, L.ERR_INVALID_ARG), ({"K": 192}, L.ERR_SHAPE), ({"N": 24}, L.ERR_SHAPE),
    ({"src": L.W_MXFP4_TILED, "n": 8}, L.ERR_SHAPE), ({"w": FAKE + 4}, L.ERR_ALIGNMENT),
])
def test_pack_arguments(kw, status):
    d = dict(src=L.W_MXFP4, w=FAKE, sc=FAKE, n=16, K=256, dst=L.W_MXFP4_TILED, N=32, row0=0) | kw
    assert L.lib().bz_pack_tiled(d["src"], d["w"], d["sc"], d["n"], d["K"], 128, d["dst"], FAKE, d["N"], d["row0"],
                                 None) == status


# ---- refusals of the Python layer ---------------------------------------------------------------------


@pytest.mark.parametrize("call", [
    lambda: mx.quantize_mx(torch.zeros(2, 64)),
    lambda: mx.dequantize_mx(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)),
    lambda: mx.mx_rows(torch.zeros(2, 128)),
    lambda: mx.mx_linear(torch.zeros(2, 128), torch.zeros(1280, dtype=torch.uint8), 16),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()


def test_element_types():
    for f in (mx.quantize_mx, mx.mx_rows):
        with pytest.raises(ValueError, match="e2m1"):
            f(torch.zeros(2, 128), "e3m2")


def test_module_arguments():
    with pytest.raises(ValueError, match="bias-free"):
        M4.Mxfp4Linear(nn.Linear(128, 16))
    with pytest.raises(ValueError, match="act_bits"):
        M4.Mxfp4Linear(nn.Linear(128, 16, bias=False), act_bits=6)
    with pytest.raises(ValueError, match="act_bits"):
        M4.quantize_module_mxfp4(nn.Sequential(), act_bits=5)
    assert M4.padded_shape(100, 2000) == (112, 2048) and M4.padded_shape(16, 128) == (16, 128)
    assert M4.tiled_shape(100, 2000) == (7, 16 * 1024 + 1024)


def _shell(n, k, act_bits=16):
    m = M4.Mxfp4Linear.__new__(M4.Mxfp4Linear)
    nn.Module.__init__(m)
    m.out_features, m.in_features, m.act_bits = n, k, act_bits
    m.register_buffer("weight_mxfp4", torch.randint(0, 255, M4.tiled_shape(n, k), dtype=torch.uint8))
    return m


class _Net(nn.Module):
    def __init__(self, a, b):
        super().__init__()
        self.a, self.b = a, b


def test_checkpoint_round_trip_and_refusals(tmp_path):
    net = _Net(_shell(48, 256, 8), _shell(50, 200))
    man = Q.save_quantized(net, tmp_path, {}, source="synthetic")
    assert man["modules"]["a"] == {"kind": "mxfp4", "layout": M4.LAYOUT_TILED, "in_features": 256, "out_features": 48,
                                   "act_bits": 8, "shapes": {"weight_mxfp4": [3, 2048 + 256]}}
    fresh = _Net(nn.Linear(256, 48, bias=False), nn.Linear(200, 50, bias=False))
    Q.install_shells(fresh, Q.read_manifest(tmp_path), "cpu")
    assert Q.load_quantized_state(fresh, tmp_path, "cpu")["missing"] == 0
    assert fresh.a.act_bits == 8 and fresh.b.act_bits == 16 and fresh.b.out_features == 50
    assert torch.equal(fresh.a.weight_mxfp4, net.a.weight_mxfp4) and torch.equal(fresh.b.weight_mxfp4, net.b.weight_mxfp4)
    for key, value, match in (("layout", "other", "layout"), ("act_bits", 3, "act_bits"), ("out_features", 64, "do not match"),
                              ("shapes", {"weight_mxfp4": [3, 2048]}, "do not match")):
        bad = Q.read_manifest(tmp_path)
        bad["modules"]["a"][key] = value
        with pytest.raises(ValueError, match=match):
            Q.install_shells(_Net(None, None), bad, "cpu")


def test_fused_weight_refuses_padded_modules():
    with pytest.raises(ValueError, match="padding"):
        FK.FusedWeight.from_mxfp4(_shell(50, 256))
    with pytest.raises(ValueError, match="padding"):
        FK.FusedWeight.from_mxfp4(_shell(48, 200))
    with pytest.raises(ValueError, match="in_features"):
        FK.FusedWeight.from_mxfp4(_shell(48, 256), _shell(48, 128))


def test_weight_buffers_are_checked():
    w = torch.zeros(1280, dtype=torch.uint8)
    G._check_weight(w, G.W_MXFP4_TILED, 16, 128, 128, None, None)
    with pytest.raises(ValueError, match="holds"):
        G._check_weight(w[:-1], G.W_MXFP4_TILED, 16, 128, 128, None, None)
    with pytest.raises(ValueError, match="sc0"):
        G._check_weight(w[:1024], G.W_MXFP4, 16, 128, 128, torch.zeros(63, dtype=torch.uint8), None)


def test_the_binding_leaves_what_it_does_not_take(monkeypatch, tmp_path):
    b = L.binding()
    cpu = torch.zeros(2, 64, dtype=torch.bfloat16)
    for args in ((), (cpu,), (cpu, "e2m1"), (None, "e2m1"), (1, 2, 3)):
        assert b.quantize_mx(*args) is None
    assert b.dequantize_mx(cpu, cpu, "e2m1", torch.bfloat16) is None
    assert b.gemv({}, {}, None, cpu, cpu, 10, 16, None, 1e-6, 0, None, torch.bfloat16) is None
    assert b.gemv(*[None] * 12) is None and b.gemv() is None
    assert b.mx_linear({}, None, cpu, cpu, 16, "e2m1", None, torch.bfloat16) is None
    assert b.mx_linear(*[None] * 8) is None
    with pytest.raises(TypeError):
        b.bind(1)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        mx.quantize_mx(cpu)
    monkeypatch.setattr(L, "_binding", None)
    monkeypatch.setattr(L, "BINDING_PATH", tmp_path / "none.so")
    with pytest.raises(RuntimeError, match="missing"):
        L.binding()
