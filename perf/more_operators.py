"""Operators over microscaled 4-bit weights, as measurable cases.

A microscaled tensor keeps, for each 32 consecutive values of a row, 4-bit (e2m1) or 8-bit (e4m3) floating-point elements
and one power of two.  Three operators work on such tensors, beside the int4, fp8 and bf16 linears of the framework:

``quantise``  rows of activations or weights to elements and scales, and the values they stand for read back
``linear``    bf16 rows times a 4-bit weight: a decode step (RMSNorm before it, SiLU gate or residual behind it), the
              rows of drafted tokens with guidance, a prompt
``mx``        the same product with the rows quantised to blocks as well, so that it runs on the matrix cores' own
              block-scaled arithmetic: prompts, and the steps of many requests

Shapes are those of the served model's layers (hidden sizes 2560, 2048 and 1024; MLPs 10240, 6144 and 8192) and of generic
ones.  Rows, shape and epilogue of a case come from the case, values from the seed.
"""

import functools
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
BLOCK = 32
# largest exponent, mantissa bits, smallest exponent and largest value of the element types
ELEMS = {"e2m1": (2, 1, 0, 6.0), "e4m3": (8, 3, -6, 448.0)}


def listed():
    return [
        # the activations of one request's step with guidance: the smallest call there is
        {"name": "quantise_b2", "kind": "quantise", "M": 2, "K": 2560, "elem": "e2m1", "dtype": "bf16", "pad": 0},
        # a weight of the backbone's MLP at load time, from its fp32 master copy
        {"name": "quantise_weight", "kind": "quantise", "M": 10240, "K": 2560, "elem": "e2m1", "dtype": "f32", "pad": 0},
        # a long prompt's MLP activations in 8 bits, columns of a wider tensor, an odd number of rows
        {"name": "quantise_prompt_e4m3", "kind": "quantise", "M": 2011, "K": 10240, "elem": "e4m3", "dtype": "bf16",
         "pad": 64},
        # depth decoder's attention output, one request: a weight that the caches hold
        {"name": "linear_o_b1", "kind": "linear", "M": 1, "N": 1024, "K": 2048, "epi": "residual", "norm": False},
        # backbone's gate and up projection of a step, norm before and SiLU gate behind it
        {"name": "linear_gate_up_b1", "kind": "linear", "M": 1, "N": 20480, "K": 2560, "epi": "silu", "norm": True},
        # the down projection of the same step with guidance
        {"name": "linear_down_b2", "kind": "linear", "M": 2, "N": 2560, "K": 10240, "epi": "residual", "norm": False},
        # 13 rows of drafted tokens through the query, key and value projections
        {"name": "linear_qkv_b13", "kind": "linear", "M": 13, "N": 6144, "K": 2560, "epi": "none", "norm": False},
        # a prompt of ordinary length on bf16 activations
        {"name": "linear_prompt_203", "kind": "linear", "M": 203, "N": 10240, "K": 2560, "epi": "none", "norm": False},
        # a step of five requests, activations in 8 bits
        {"name": "mx_step_b5_e4m3", "kind": "mx", "M": 5, "N": 2560, "K": 10240, "epi": "residual", "elem": "e4m3"},
        # an ordinary prompt, activations in 4 bits
        {"name": "mx_prompt_611", "kind": "mx", "M": 611, "N": 10240, "K": 2560, "epi": "none", "elem": "e2m1"},
        # a long prompt's down projection, activations in 8 bits
        {"name": "mx_prompt_2011_e4m3", "kind": "mx", "M": 2011, "N": 2560, "K": 10240, "epi": "residual",
         "elem": "e4m3"},
        # the prompts of several requests at once through the gate and up projections, activations in 4 bits
        {"name": "mx_prompts_8192", "kind": "mx", "M": 8192, "N": 20480, "K": 2560, "epi": "none", "elem": "e2m1"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantise", "linear", "linear", "mx", "mx"])
    if kind == "quantise":
        k = BLOCK * _spread(rng, 1, 640)
        return {"kind": kind, "M": _spread(rng, 1, min(16384, 26_000_000 // k)), "K": k,
                "elem": rng.choice(["e2m1", "e4m3"]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "pad": rng.choice([0, 0, 8, 1000])}
    if rng.random() < 0.5:
        n, k = rng.choice([(2048, 2048), (6144, 2048), (12288, 2048), (2048, 6144), (4096, 2560), (2560, 4096),
                           (20480, 2560), (2560, 10240), (16384, 1024), (1024, 8192)])
    else:
        n, k = 16 * _spread(rng, 4, 1024), 128 * _spread(rng, 1, 80)
    case = {"kind": kind, "M": _spread(rng, 1, 40) if rng.random() < 0.5 else _spread(rng, 33, 2048), "N": n, "K": k}
    if kind == "mx":
        return case | {"epi": rng.choice(["none", "residual"]), "elem": rng.choice(["e2m1", "e4m3"])}
    if case["M"] > 32:  # prompts: no norm, no epilogue
        return case | {"epi": "none", "norm": False}
    case["epi"] = rng.choice(["none", "residual", "silu"])
    # the norm stands before the projections of a layer's input, the residual behind those of its output
    return case | {"norm": case["M"] <= 8 and case["epi"] != "residual" and rng.random() < 0.6}


def work(case):
    m, k = case["M"], case["K"]
    if case["kind"] == "quantise":
        held = m * k // (2 if case["elem"] == "e2m1" else 1) + m * k // BLOCK
        # in, held elements and scales written and read again, the values read back
        return {"bytes": m * k * (4 if case["dtype"] == "f32" else 2) + 2 * held + m * k * 2, "flops": 4 * m * k}
    n = case["N"]
    n_out = n // 2 if case["epi"] == "silu" else n
    out = m * n_out * 2 * (2 if case["epi"] == "residual" else 1)
    return {"bytes": n * k // 2 + n * k // BLOCK + m * k * 2 + out + (2 * k if case.get("norm") else 0),
            "flops": 2 * m * n * k}


# ---- what a program has in hand before the call ----------------------------------------------------


@functools.lru_cache(maxsize=None)
def _own():
    sys.path.insert(0, os.path.join(os.getcwd(), "breeze-tts-2_amd"))
    from breeze_amd import gemv, mx

    return gemv, mx


def _activations(g, m, k):
    """Rows as a layer's input has them: a spread of channel sizes, a few channels far above the rest."""
    size = torch.exp(0.5 * torch.randn(k, device=DEV, generator=g))
    size[torch.rand(k, device=DEV, generator=g) < 0.004] *= 20
    return torch.randn(m, k, device=DEV, generator=g) * size


def _weight(g, n, k):
    """Codes (two to a byte, the even k low) and scales of a random weight."""
    codes = torch.empty(n, k // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(n, k // BLOCK, dtype=torch.uint8, device=DEV)
    for lo in range(0, n, 4096):
        hi = min(n, lo + 4096)
        v, s = _round_blocks(torch.randn(hi - lo, k, device=DEV, generator=g) * k ** -0.5, "e2m1")
        v = v * ((254 - s.int()) << 23).view(F32).repeat_interleave(BLOCK, -1)  # the elements themselves
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
        c = torch.bucketize(v.abs(), grid) + 8 * (v < 0)
        codes[lo:hi], scales[lo:hi] = (c[:, ::2] + 16 * c[:, 1::2]).to(torch.uint8), s
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    m, k = case["M"], case["K"]
    s = {"case": case}
    if case["kind"] == "quantise":
        dt = {"bf16": BF16, "f16": torch.float16, "f32": F32}[case["dtype"]]
        s["x"] = _activations(g, m, k + case["pad"]).to(dt)[:, :k]
        return s
    n = case["N"]
    s["x"] = _activations(g, m, k).to(BF16)
    s["codes"], s["scales"] = _weight(g, n, k)
    s["gamma"] = (1 + 0.1 * torch.randn(k, device=DEV, generator=g)).to(BF16) if case.get("norm") else None
    s["res"] = torch.randn(m, n, device=DEV, generator=g).to(BF16) if case["epi"] == "residual" else None
    if own:  # a program lays a weight out once, when it loads it
        gemv, _ = _own()
        s["fmt"] = gemv.W_MXFP4_TILED_PAIRED if case["epi"] == "silu" else gemv.W_MXFP4_TILED
        s["w"] = gemv.pack_tiled(gemv.W_MXFP4, s["codes"], k, s["fmt"], sc0=s["scales"])
    return s


# ---- one pass ---------------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if not own:
        return _plain_quantise(s) if case["kind"] == "quantise" else _plain_product(s)
    gemv, mx = _own()
    if case["kind"] == "quantise":
        codes, scales = mx.quantize_mx(s["x"], case["elem"])
        return mx.dequantize_mx(codes, scales, case["elem"]), scales
    if case["kind"] == "mx":
        return mx.mx_linear(s["x"], s["w"], case["N"], elem=case["elem"], residual=s["res"])
    if case["M"] > 32:
        return gemv.dequant_matmul(s["x"], s["w"], s["fmt"], case["N"], case["K"])
    epi = {"none": gemv.EPI_NONE, "residual": gemv.EPI_RESIDUAL, "silu": gemv.EPI_SILU_GATE}[case["epi"]]
    return gemv.gemv(s["x"], s["w"], s["fmt"], case["N"], gamma=s["gamma"], eps=EPS, epilogue=epi, residual=s["res"])


def _round_blocks(x, elem):
    """The values that x's blocks stand for (fp32) and the scale codes (uint8)."""
    emax, bits, emin, top = ELEMS[elem]
    v = x.float().unflatten(-1, (-1, BLOCK))
    amax = v.abs().amax(-1, keepdim=True)
    # floor(log2 amax) + 127 is the exponent field of the fp32 amax
    code = ((amax.view(torch.int32) >> 23) - emax).clamp(min=1)
    scale = (code << 23).view(F32)
    v = v * ((254 - code) << 23).view(F32)
    # a step of the element type at v: ties go to the even multiple, which is the even code
    step = (((v.abs().view(torch.int32) >> 23).clamp(min=emin + 127) - bits) << 23).view(F32)
    v = (torch.round(v / step) * step).clamp(-top, top) * scale
    return v.flatten(-2), code.squeeze(-1).to(torch.uint8)


def _plain_quantise(s):
    v, code = _round_blocks(s["x"], s["case"]["elem"])
    return v.to(BF16), code  # (bf16 holds every such value)


def _values(codes, scales):
    """fp32 weight [N, K] from codes and scales."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    table = torch.cat([table, -table])
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(-2)
    return v * (scales.int() << 23).view(F32).repeat_interleave(BLOCK, -1)


def _plain_product(s):
    case = s["case"]
    x = s["x"].float()
    if case["kind"] == "mx":
        x, _ = _round_blocks(x, case["elem"])
    rstd = 1.0
    if s["gamma"] is not None:
        rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        x = (x * s["gamma"].float()).to(BF16).float()  # the operator's own rounding, as the bf16 linears define it
    n, m = case["N"], case["M"]
    y = torch.empty(m, n, device=DEV)
    for lo in range(0, n, 8192):  # a run of rows of the weight at a time: its 64-bit indices are large
        y[:, lo:lo + 8192] = x @ _values(s["codes"][lo:lo + 8192], s["scales"][lo:lo + 8192]).T
    y = y * rstd
    if case["epi"] == "silu":
        gate, up = y[:, : n // 2], y[:, n // 2:]
        y = gate / (1 + torch.exp(-gate)) * up
    elif case["epi"] == "residual":
        y = y + s["res"].float()
    return y.to(BF16)


# ---- the definition, in 64 bits ------------------------------------------------------------------------


def _grid(elem):
    """The values of the element type from 0 up; a value's place is its code."""
    emax, bits, emin, top = ELEMS[elem]
    values = [i * 2.0 ** (emin - bits) for i in range(2 ** bits)]  # the subnormal ones
    values += [2.0 ** e * (1 + i / 2 ** bits) for e in range(emin, emax + 1) for i in range(2 ** bits)]
    return torch.tensor([v for v in values if v <= top], dtype=F64, device=DEV)


def _pow2(e):
    """2^e of whole numbers e, exactly: exp2 and pow are free to be a rounding off."""
    return ((e.long() + 1023) << 52).view(F64)


def _exact_blocks(x, elem):
    grid = _grid(elem)
    x = x.double().unflatten(-1, (-1, BLOCK))
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax).exponent - 1 - ELEMS[elem][0]
    e = torch.where(amax > 0, e, -126).clamp(min=-126)
    y = x / _pow2(e)
    # the two neighbours on the grid, the nearer one, the even code where they are as near
    hi = torch.bucketize(y.abs(), grid).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    to_lo, to_hi = y.abs() - grid[lo], grid[hi] - y.abs()
    q = torch.where((to_lo < to_hi) | ((to_lo == to_hi) & (lo % 2 == 0)), lo, hi)
    return (grid[q] * y.sign() * _pow2(e)).flatten(-2), (e + 127).squeeze(-1).to(torch.uint8)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantise":
        return _exact_blocks(s["x"], case["elem"])
    x = s["x"].double()
    if case["kind"] == "mx":
        x, _ = _exact_blocks(x, case["elem"])
    rstd = 1.0
    if s["gamma"] is not None:
        rstd = (x.square().mean(-1, keepdim=True) + EPS) ** -0.5
        x = (s["x"] * s["gamma"]).double()  # bf16: the definition rounds the weighted input
    sign_grid = torch.cat([_grid("e2m1"), -_grid("e2m1")])
    y = torch.empty(case["M"], case["N"], dtype=F64, device=DEV)
    for lo in range(0, case["N"], 2048):
        c = s["codes"][lo:lo + 2048]
        w = torch.stack([sign_grid[(c % 16).int()], sign_grid[(c // 16).int()]], -1).flatten(-2)
        w = w.unflatten(-1, (-1, BLOCK)) * _pow2(s["scales"][lo:lo + 2048].int() - 127)[..., None]
        y[:, lo:lo + 2048] = x @ w.flatten(-2).T
    y = y * rstd
    if case["epi"] == "silu":
        gate, up = y.chunk(2, -1)
        return gate * torch.sigmoid(gate) * up
    return y + s["res"].double() if case["epi"] == "residual" else y
