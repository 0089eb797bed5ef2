"""Microscaled 4-bit (MXFP4) weight Linear, on MI355X.

The third quantized module beside Int4Linear and Fp8Linear, with the same
constructor, forward() contract and module swap (no counterpart in the
reference, whose weights are int4 or fp8: models/int4_linear.py,
models/fp8_linear.py).  A weight takes 4.25 bits a value: e2m1 elements and one
power of two for each 32 (mx.py).

``weight_mxfp4`` holds the tiled layout (LAYOUT_TILED, the bytes of
BZ_W_MXFP4_TILED in include/bz_gemv.h): uint8 [N'/16, bytes per 16-row block],
N' and K' the features rounded up to 16 rows and 128 columns.  The added rows
and columns are zeros: calls pad x with zeros and drop the added outputs.

Calls of up to PREFILL_ROWS rows read the activations in bf16, as Int4Linear
and Fp8Linear do: a decode step is bound by the weight's bytes.  Longer ones
(a prompt) are bound by the matrix cores, and ``act_bits`` says what they
multiply: 16, the bf16 activations; 8 or 4, activations quantised to
microscaled blocks (e4m3 or e2m1) on the way, at the matrix cores' 8- or 4-bit
rate, and without a gradient.
"""

from __future__ import annotations

import torch
from torch import nn

from ._swap import swap_linears
from .gemv import W_MXFP4, W_MXFP4_TILED, dequant_matmul, gemv, pack_tiled, tiled_bytes
from .mx import BLOCK, followed, mx_linear, quantize_mx

MIN_QUANT_BYTES = 8 * 1024 * 1024

DEFAULT_TARGET_NAMES = ("gate_proj", "up_proj", "down_proj")

# Above this many rows a call is a prefill (as in int4_linear.py).
PREFILL_ROWS = 32

# Tag recorded by the checkpoint manifest.
LAYOUT_TILED = "bz-mxfp4-tiled16-v1"

_ACT_ELEM = {4: "e2m1", 8: "e4m3"}


def padded_shape(out_features: int, in_features: int) -> tuple[int, int]:
    """Rows and columns a weight of this shape is stored with."""
    return -(-out_features // 16) * 16, -(-in_features // 128) * 128


def tiled_shape(out_features: int, in_features: int) -> tuple[int, int]:
    """uint8 shape of weight_mxfp4: [N'/16, bytes per 16-row block]."""
    n, k = padded_shape(out_features, in_features)
    return n // 16, tiled_bytes(W_MXFP4_TILED, 16, k)


def quantize_mxfp4(weight: torch.Tensor) -> torch.Tensor:
    """weight [N, K] (bf16, fp16 or fp32) -> weight_mxfp4, on the device the weight lives on
    (a CPU weight is quantized on the current GPU and the result moved back)."""
    n, k = weight.shape
    weight = weight.detach()  # (a parameter is quantized as it is)
    w = weight if weight.device.type == "cuda" else weight.to(torch.device("cuda", torch.cuda.current_device()))
    if w.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        w = w.float()
    n_pad, k_pad = padded_shape(n, k)
    if (n_pad, k_pad) != (n, k):
        w = torch.nn.functional.pad(w, (0, k_pad - k, 0, n_pad - n))
    codes, scales = quantize_mx(w, "e2m1")
    tiled = pack_tiled(W_MXFP4, codes, k_pad, W_MXFP4_TILED, sc0=scales).view(*tiled_shape(n, k))
    return tiled if weight.device.type == "cuda" else tiled.to(weight.device)


def _product(x: torch.Tensor, w: torch.Tensor, n: int, act_bits: int) -> torch.Tensor:
    """x [M, K] bf16 times a weight of n rows, in the way of its row count; a call
    that autograd follows, backward or forward, goes the way of the prompts,
    which it can follow."""
    if x.shape[0] <= PREFILL_ROWS and not followed(x):
        return gemv(x, w, W_MXFP4_TILED, n)
    if act_bits == 16:
        return dequant_matmul(x, w, W_MXFP4_TILED, n, x.shape[1])
    return mx_linear(x, w, n, elem=_ACT_ELEM[act_bits])


@torch.library.custom_op("breeze_amd::mxfp4_linear", mutates_args=())
def mxfp4_linear_op(x: torch.Tensor, w: torch.Tensor, n: int, act_bits: int) -> torch.Tensor:
    """_product where torch.compile traces: the row count decides when the call
    runs, so a compiled prompt multiplies what an eager one does."""
    return _product(x, w, n, act_bits)


@mxfp4_linear_op.register_fake
def _mxfp4_linear_fake(x, w, n, act_bits):
    return x.new_empty((x.shape[0], n), dtype=torch.bfloat16)


class Mxfp4Linear(nn.Module):
    """Drop-in replacement for a bias-free nn.Linear using microscaled 4-bit weights."""

    def __init__(self, linear: nn.Linear, act_bits: int = 16, device: torch.device | str | None = None) -> None:
        super().__init__()
        if linear.bias is not None:
            raise ValueError("Mxfp4Linear expects a bias-free Linear")
        if act_bits not in (4, 8, 16):
            raise ValueError(f"act_bits must be 4, 8 or 16, got {act_bits}")
        weight = linear.weight.data if device is None else linear.weight.data.to(device)
        self.out_features, self.in_features = (int(d) for d in weight.shape)
        self.act_bits = act_bits
        self.register_buffer("weight_mxfp4", quantize_mxfp4(weight))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape = x.shape
        flat = x if x.dim() == 2 else x.reshape(-1, shape[-1])
        w, n, k = self.weight_mxfp4, self.out_features, self.in_features
        n_pad, k_pad = padded_shape(n, k)
        if flat.dtype != torch.bfloat16:
            flat = flat.to(torch.bfloat16)
        if k_pad != k:
            flat = torch.nn.functional.pad(flat, (0, k_pad - k))
        if torch.compiler.is_compiling():
            out = torch.ops.breeze_amd.mxfp4_linear(flat, w, n_pad, self.act_bits)
        else:
            out = _product(flat, w, n_pad, self.act_bits)
        if n_pad != n:
            out = out[:, :n].contiguous()
        if x.dtype != torch.bfloat16:
            out = out.to(x.dtype)
        return out if x.dim() == 2 else out.reshape(*shape[:-1], n)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, mxfp4=True, block={BLOCK}, "
                f"act_bits={self.act_bits}")


def quantize_module_mxfp4(
    root: nn.Module,
    *,
    target_names: tuple[str, ...] = DEFAULT_TARGET_NAMES,
    min_bytes: int = MIN_QUANT_BYTES,
    device: torch.device | str | None = None,
    act_bits: int = 16,
) -> dict[str, int]:
    """Swap qualifying Linear layers under ``root`` for MXFP4 equivalents, with the
    counting rules and stats of quantize_module_int4.  Saved bytes: 4.25 of a
    bf16 weight's 16 bits stay."""
    if act_bits not in (4, 8, 16):
        raise ValueError(f"act_bits must be 4, 8 or 16, got {act_bits}")
    st = swap_linears(
        root,
        target_names,
        min_bytes,
        build=lambda lin: Mxfp4Linear(lin, act_bits=act_bits, device=device),
        saved_bytes=lambda nbytes: nbytes - nbytes * 17 // 64,
        tolerate_errors=False,
        drop_original=True,
    )
    return {
        "converted": st.converted,
        "skipped_below_threshold": st.small,
        "weight_bytes_saved": st.saved,
    }
