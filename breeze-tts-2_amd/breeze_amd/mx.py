"""Operators over microscaled blocks (include/bz_mx.h).

A microscaled tensor keeps, for each 32 consecutive values of a row, elements
of a narrow floating-point type and one power of two:

``quantize_mx``    rows to elements and scale codes, the layout checkpoints hold
``dequantize_mx``  the values they stand for
``mx_rows``        rows to the operand order of the matrix cores, for several
                   ``mx_linear`` over the same rows
``mx_linear``      rows, quantised to blocks, times a 4-bit weight on the matrix
                   cores' block-scaled arithmetic

Element types ("elem"): "e2m1" (4 bits, 0 0.5 1 1.5 2 3 4 6) and "e4m3" (OCP
FP8, up to 448).  A block with largest magnitude a has the scale
2^max(floor(log2 a) - emax, -126), emax 2 or 8, stored as the exponent plus 127
in a byte; each element is its value over the scale, rounded to the nearest
(ties to the even code), magnitudes above the type's largest to the largest.
A block that holds a NaN or an infinity has the code 255 and reads back as NaN.

Weights are e2m1: ``quantize_mx`` of an [N, K] weight, laid out for the kernels
by ``gemv.pack_tiled(W_MXFP4, codes, K, W_MXFP4_TILED, sc0=scales)``.  bf16 rows
times such a weight, with nothing quantised on the way, are ``gemv.gemv`` and
``gemv.dequant_matmul``; ``mxfp4_linear.Mxfp4Linear`` is the module.

Calls follow torch's current stream of the tensors' device, do not synchronise,
and may be captured into graphs and made from several streams at once.  None of
them has a gradient: rows, a residual or an ``out`` that autograd follows,
backward or forward, are refused.
"""

from __future__ import annotations

import functools
from typing import Optional, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import DT_BF16, DT_F32, MX_E2M1, MX_E4M3, MX_F16, MX_ROWS, MX_TILED, W_MXFP4_TILED

__all__ = ["BLOCK", "MxRows", "quantize_mx", "dequantize_mx", "mx_rows", "mx_linear"]

BLOCK = 32

# Up to this many rows mx_linear is one launch over the rows themselves; not for
# more than 16 rows over a weight of more than ONE_ROUND rows, which takes a second
# round of workgroups of eight row blocks, each quantising x (N40960 K2560 M = 17 e2m1
# 22.6 us, two launches 18.6; N151936 72.3 and 48.7 for 32; N28672 K4096 17.4 and 21.9 for
# 17, 19.7 and 19.7 for 32; N32768 K2560 13.9 and 16.3, 15.7 and 15.3).
FEW_ROWS = 32
ONE_ROUND = 32768

_ELEM = {"e2m1": MX_E2M1, "e4m3": MX_E4M3}
_X = {torch.bfloat16: DT_BF16, torch.float32: DT_F32, torch.float16: MX_F16}
_OUT = {torch.bfloat16: DT_BF16, torch.float32: DT_F32}


def _elem(elem: str) -> int:
    code = _ELEM.get(elem)
    if code is None:
        raise ValueError(f"elem must be 'e2m1' or 'e4m3', got {elem!r}")
    return code


def _gpu(name: str, t: torch.Tensor, index: int) -> None:
    at = t.get_device()  # -1 on the CPU
    if at < 0:
        raise RuntimeError(f"{name} must be a GPU tensor (got {t.device}); the HIP path has no CPU fallback")
    if at != index:
        raise RuntimeError(f"{name} is on {t.device}, expected cuda:{index}")


def followed(t: torch.Tensor) -> bool:
    """Whether autograd follows t, backward or forward."""
    if t.requires_grad and torch.is_grad_enabled():
        return True
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _no_grad(what: str, *tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and followed(t):
            raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on x.detach()")


def _call(index: int, f, *args) -> None:
    """f(*args, stream) on the device's current stream, with the device current."""
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = f(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = f(*args, stream)
    if rc:
        raise _lib.BzError(rc, f.__name__)


def _counted(M: int, K: int) -> None:
    """The library counts rows and columns in 32 bits (ctypes would cut them to that)."""
    if M >= 1 << 31 or K >= 1 << 31:
        raise ValueError(f"{M} rows of {K} columns: both have to be below 2^31")


def _rows(x: torch.Tensor, unit: int) -> tuple:
    """(x with rows the kernels can read, M, K, row stride, type code, device
    index)."""
    index, shape, dt = x.get_device(), x.shape, _X.get(x.dtype)
    if index < 0:
        _gpu("x", x, index)
    if len(shape) != 2:
        raise ValueError(f"x must be [rows, columns], got {list(shape)}")
    if dt is None:
        raise TypeError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    M, K = shape
    if K < 1 or K % unit:
        raise ValueError(f"{K} columns are not a positive multiple of {unit}")
    _counted(M, K)
    ld, inner = x.stride()
    if M <= 1:
        ld = K
    if inner != 1 or ld < K:  # a transposed matrix, an expanded row
        x, ld = x.contiguous(), K
    return x, M, K, ld, dt, index


def quantize_mx(x: torch.Tensor, elem: str = "e2m1") -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of x [M, K] (bf16, fp16 or fp32; K a multiple of 32):
    codes uint8 [M, K/2] with the even column in the low half (e2m1) or
    float8_e4m3fn [M, K]; scales uint8 [M, K/32]."""
    if x.is_cuda:  # nothing to convert: checked and made in C++
        held = (_lib._binding or _lib.binding()).quantize_mx(x, elem)
        if held is not None:
            return held
    code = _elem(elem)
    _no_grad("quantize_mx", x)
    x, M, K, ld, dt, index = _rows(x, BLOCK)
    if code == MX_E2M1:
        codes = torch.empty((M, K // 2), dtype=torch.uint8, device=x.device)
    else:
        codes = torch.empty((M, K), dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((M, K // BLOCK), dtype=torch.uint8, device=x.device)
    if M:
        _call(index, _lib.lib().bz_mx_quantize, x.data_ptr(), dt, ld, M, K, code, MX_ROWS, codes.data_ptr(),
              scales.data_ptr())
    return codes, scales


def dequantize_mx(codes: torch.Tensor, scales: torch.Tensor, elem: str = "e2m1",
                  dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [M, K] (bf16 or fp32) that quantize_mx's codes and scales stand
    for: exact, in bf16 down to 2^-126."""
    if codes.is_cuda:
        out = (_lib._binding or _lib.binding()).dequantize_mx(codes, scales, elem, dtype)
        if out is not None:
            return out
    code, index, shape = _elem(elem), codes.get_device(), codes.shape
    if index < 0 or scales.get_device() != index:
        _gpu("codes", codes, index)
        _gpu("scales", scales, index)
    dt = _OUT.get(dtype)
    if dt is None:
        raise TypeError(f"values are bfloat16 or float32, not {dtype}")
    if len(shape) != 2 or scales.dtype is not torch.uint8 or not (
            codes.dtype is torch.uint8 or code == MX_E4M3 and codes.dtype is torch.float8_e4m3fn):
        raise ValueError("codes must be 2-D, uint8 (or float8_e4m3fn for e4m3), and scales uint8")
    M, K = shape
    if code == MX_E2M1:
        K *= 2
    if K < 1 or K % BLOCK or scales.shape != (M, K // BLOCK):
        raise ValueError(f"codes {list(shape)} and scales {list(scales.shape)} are not those of {elem} rows")
    _counted(M, K)
    if not codes.is_contiguous() or codes.data_ptr() % 4:
        codes = codes.clone(memory_format=torch.contiguous_format)
    if not scales.is_contiguous():
        scales = scales.contiguous()
    out = torch.empty((M, K), dtype=dtype, device=codes.device)
    if M:
        _call(index, _lib.lib().bz_mx_dequantize, codes.data_ptr(), scales.data_ptr(), code, M, K, out.data_ptr(), dt, K)
    return out


class MxRows:
    """Quantised rows in the operand order of the matrix cores (mx_rows)."""

    __slots__ = ("data", "shape", "elem")

    def __init__(self, data: torch.Tensor, shape: tuple[int, int], elem: str):
        self.data, self.shape, self.elem = data, shape, elem


@functools.lru_cache(maxsize=4096)
def _rows_bytes(elem: int, M: int, K: int) -> int:
    return int(_lib.lib().bz_mx_rows_bytes(elem, M, K))


def mx_rows(x: torch.Tensor, elem: str = "e2m1") -> MxRows:
    """x [M, K] (bf16, fp16 or fp32; K a multiple of 128) quantised to blocks,
    for mx_linear: once for all products that read the same rows."""
    code = _elem(elem)
    x, M, K, ld, dt, index = _rows(x, 128)
    _no_grad("mx_rows", x)
    return MxRows(_tiled_rows(x, M, K, ld, dt, code, index), (M, K), elem)


def _tiled_rows(x, M: int, K: int, ld: int, dt: int, code: int, index: int) -> torch.Tensor:
    data = torch.empty(_rows_bytes(code, M, K), device=x.device, dtype=torch.uint8)
    if M:
        _call(index, _lib.lib().bz_mx_quantize, x.data_ptr(), dt, ld, M, K, code, MX_TILED, data.data_ptr(), None)
    return data


# Workspaces of products that slice K: one for each device and stream, and for
# each graph capture under way.
_WS: dict = {}
_WS_RETIRED: list = []
# (element type, M, n, K) -> _plan's answer and the bytes of the quantised rows, for
# the binding.  Forgotten when there are too many: a server that sees prompts of
# every length adds one for each of them and each weight.
_PLANS: dict = {}
_MOST_PLANS = 4096
_NO_WAY = (1 << 64) - 1  # what bz_mx_gemv_workspace gives for a shape it does not take


@functools.lru_cache(maxsize=4096)
def _plan(elem: int, M: int, n: int, k: int, cfg: int, rows: bool) -> tuple[int, bool, int]:
    """(bytes of the weight, whether one launch over bf16 rows takes the shape,
    workspace bytes)."""
    lib = _lib.lib()
    weight = 0 < n < 1 << 31 and int(lib.bz_tiled_bytes(W_MXFP4_TILED, n, k)) or -1
    if rows and 0 < M <= FEW_ROWS and (M <= 16 or n <= ONE_ROUND or cfg):
        need = int(lib.bz_mx_gemv_workspace(elem, M, n, k, cfg))
        if need != _NO_WAY or cfg:  # (a forced shape it does not take is refused by the call)
            return weight, True, 0 if need == _NO_WAY else need
    return weight, False, int(lib.bz_mx_gemm_workspace(elem, M, n, k, cfg))


def mx_linear(x: Union[torch.Tensor, MxRows], w: torch.Tensor, n: int, *, elem: str = "e2m1",
              residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
              out_dtype: torch.dtype = torch.bfloat16, cfg: int = 0) -> torch.Tensor:
    """q(x) @ w_eff^T (+ residual) -> [M, n]: x [M, K] (bf16, fp16 or fp32), quantised to
    blocks of ``elem`` on the way, or the MxRows of it; w a W_MXFP4_TILED weight of n
    rows and K columns.  e2m1 products are exact and their sums fp32; e4m3's are
    first added by eights on the matrix core's grid (include/bz_mx.h), which leaves
    an fp32 result 2e-5 of its norm off, bf16's rounding being 1.7e-3.  The result
    is rounded once, to out's dtype (bf16 or fp32).  residual: [M, n] bf16 or fp32,
    may be out itself; out: [M, n] with unit column stride, apart from x and w.
    cfg: a launch shape (include/bz_mx.h) instead of the built-in rule's.

    Few rows are for a step that has to round its activations as the prompt
    before it did; gemv.gemv over the same weight rounds none and takes less at one
    or two (N2560 K10240 M = 2 5.3 us against 6.9, N1024 K2048 M = 1 2.7 and 3.4)."""
    rows = isinstance(x, MxRows)
    if not (rows or cfg) and out is None and x.is_cuda:  # nothing to convert: checked and made in C++
        y = (_lib._binding or _lib.binding()).mx_linear(_PLANS, _raw_workspace, x, w, n, elem, residual, out_dtype)
        if y is not None:
            return y
    if rows:
        src, (M, K), code = x.data, x.shape, _elem(x.elem)
        index, few = src.get_device(), False
        if index < 0 or src.numel() * src.element_size() != _rows_bytes(code, M, K) or not src.is_contiguous():
            _gpu("x", src, index)
            raise ValueError(f"these are not the MxRows of {M} x {K} {x.elem} rows")
    else:
        code = _elem(elem)
        src, M, K, ld, dt, index = _rows(x, 128)
        _no_grad("mx_linear", x)
        # up to 32 rows that a launch can read as they are: quantised inside it
        few = dt == DT_BF16 and M <= FEW_ROWS and not (ld & 7 or src.data_ptr() & 15) and M * ld < 1 << 30
    _no_grad("mx_linear", residual, out)
    fits = few
    weight, few, need = _plan(code, M, n, K, cfg, few)
    if w.get_device() != index or w.numel() * w.element_size() != weight or not w.is_contiguous() or w.data_ptr() & 15:
        _gpu("w", w, index)
        raise ValueError(f"w must be a contiguous W_MXFP4_TILED weight of {n} x {K} (rows a multiple of 16), "
                         f"{max(weight, 0)} bytes, at a multiple of 16; got {w.numel() * w.element_size()}")
    if out is None:
        odt = _OUT.get(out_dtype)
        if odt is None:
            raise TypeError(f"out is bfloat16 or float32, not {out_dtype}")
        out, ldo = torch.empty((M, n), dtype=out_dtype, device=w.device), n
        fresh = True
    else:
        _gpu("out", out, index)
        odt, fresh = _OUT.get(out.dtype), False
        if odt is None or out.shape != (M, n) or (out.stride(1) != 1 and n > 1) or (M > 1 and out.stride(0) < n):
            raise ValueError(f"out must be a bf16 or fp32 [{M}, {n}] tensor whose rows are contiguous")
        for name, t in (("x", src), ("w", w)):
            if _overlap(out, t):
                raise ValueError(f"out must not overlap {name}")
        ldo = out.stride(0) if M > 1 else n
    res = rdt = ldr = 0
    if residual is not None:
        rdt = _OUT.get(residual.dtype)
        if residual.get_device() != index or rdt is None or residual.shape != (M, n):
            _gpu("residual", residual, index)
            raise ValueError(f"residual must be a bf16 or fp32 [{M}, {n}] tensor")
        ldr, inner = residual.stride()
        if (inner != 1 and n > 1) or (M > 1 and ldr < n) \
                or not (fresh or _same(out, residual) or not _overlap(out, residual)):
            residual = residual.clone(memory_format=torch.contiguous_format)
            ldr = n
        res = residual.data_ptr()
        if M <= 1:
            ldr = n
    if M == 0:
        return out
    if not cfg and not rows and fits == (M <= FEW_ROWS):  # (not the two launches of few rows that need a copy)
        if len(_PLANS) >= _MOST_PLANS:
            _PLANS.clear()
        _PLANS[code, M, n, K] = weight, few, need, 0 if few else _rows_bytes(code, M, K)
    lib, ws = _lib.lib(), 0
    if not (few or rows):
        src = _tiled_rows(src, M, K, ld, dt, code, index)
    if need:
        ws, _ = _raw_workspace(index, torch._C._cuda_getCurrentRawStream(index), need)
    if few:
        _call(index, lib.bz_mx_gemv, code, src.data_ptr(), ld, M, w.data_ptr(), n, K, res, rdt, ldr, out.data_ptr(),
              odt, ldo, ws, need, cfg)
    else:
        _call(index, lib.bz_mx_gemm, code, src.data_ptr(), M, w.data_ptr(), n, K, res, rdt, ldr, out.data_ptr(),
              odt, ldo, ws, need, cfg)
    return out


def _raw_workspace(index: int, stream: int, nbytes: int) -> tuple:
    """(address, bytes) of the workspace of products on this stream."""
    ws = _lib.stream_workspace(_WS, (index,), nbytes, torch.device("cuda", index), stream, _WS_RETIRED)
    return ws.data_ptr(), ws.numel() * 4


def _span(t: torch.Tensor) -> tuple[int, int]:
    size = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + size * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a and b may share memory; matrices of one row stride are compared
    column range by column range, as views of one wider tensor have them."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if not (a0 < b1 and b0 < a1):
        return False
    if a.dim() != 2 or b.dim() != 2 or a.stride(1) != 1 or b.stride(1) != 1:
        return True
    step, wide_a, wide_b = (a.stride(0) * a.element_size(), a.shape[1] * a.element_size(), b.shape[1] * b.element_size())
    if b.stride(0) * b.element_size() != step or max(wide_a, wide_b) > step:
        return True
    at = (b0 - a0) % step  # of b's rows, from the last start of one of a's
    return at < wide_a or at + wide_b > step


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether each element of b lies where that of a does."""
    return a.data_ptr() == b.data_ptr() and a.dtype == b.dtype and a.stride() == b.stride()
