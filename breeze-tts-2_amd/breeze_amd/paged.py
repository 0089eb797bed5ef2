"""Operators over a paged key/value cache (include/bz_paged.h).

A server that runs requests of different lengths keeps their keys and values in
pages of one pool instead of a static [B, HKV, S, D] cache each:

``paged_rope_cache``         q/k RMSNorm + RoPE of the new tokens, their keys and
                             values into the pages, rotated queries out
``paged_attention``          attention of each sequence's newest rows over its pages
``shared_prefix_attention``  the same where sequences begin with a shared prompt (a
                             voice), whose pages are stored once and read once for many rows

Common arguments:

k_pages, v_pages  [pages, HKV, page_size, D] bf16, or float8_e4m3fn with k_scale /
                  v_scale (fp32 [HKV]: a code stands for code * scale, whatever the scale's
                  sign, 0 included).  Any strides with contiguous D, so a
                  [pages, page_size, HKV, D] pool is passed as its transpose(1, 2).
                  page_size a power of two, 16 .. 4096.
block_table       int32 [B, W]: position j of sequence b lies in page
                  block_table[b, j // page_size].  Entries past a sequence's length are not
                  read; one outside [0, pages) is a page that is not there (not written,
                  not attended).
kv_lens           int32 [B], the new rows included
q_starts          int32 [B + 1]: sequence b has the rows q_starts[b] .. q_starts[b + 1] - 1,
                  its newest positions in order; None: one row each.  Rows of no sequence
                  are not touched: in a tensor that the call allocates they hold anything.
                  Starts must not decrease; if they do, rows hold anything.

Lengths, tables and starts are read on the device: no call synchronizes, and a
captured graph follows them.  Calls may run on several streams at once, and graphs on
any: each stream and each capture has a workspace of its own, for the life of the
process (1 MB for the steps of a few requests, 100 MB for 8191 rows of 16 heads of 128;
a graph clears its own once a replay).  Calls may come from several host threads: those
on one stream go one after the other, each as a whole.

Sums and softmax are in fp32.  Probabilities go into their products with the values as
two bf16 parts where the sequences (or prefixes) of a call have 32 query rows of a
key/value head or fewer on average (16 for D = 256), else rounded to one: a token's
result depends in its last bits on the company it has.
"""

from __future__ import annotations

import functools
import threading
from typing import Optional

import torch

from . import _lib
from ._lib import DT_BF16, DT_F32, KV_E4M3

__all__ = ["paged_rope_cache", "paged_attention", "shared_prefix_attention"]

# One zeroed workspace for each device and stream, and for each graph capture
# under way: the kernels leave its counters at zero.
_WS: dict[tuple, torch.Tensor] = {}
_WS_RETIRED: list = []

# One lock for each device and stream.  A call can be two launches, the second of which reads what
# the first left in the stream's workspace, and the library is called without the GIL: another
# thread's first launch between the two would overwrite it.
_LOCKS: dict[tuple, object] = {}

_KV = {torch.bfloat16: DT_BF16, torch.float8_e4m3fn: KV_E4M3}
_CS = {torch.bfloat16: DT_BF16, torch.float32: DT_F32}


def _gpu(name: str, t: torch.Tensor, index: int) -> None:
    at = t.get_device()  # -1 on the CPU
    if at == index and at >= 0:
        return
    if at < 0:
        raise RuntimeError(f"{name} must be a GPU tensor (got {t.device}); the HIP path has no CPU fallback")
    raise RuntimeError(f"{name} is on {t.device}, expected cuda:{index}")


def _ints(name: str, t: torch.Tensor, shape: tuple, index: int) -> int:
    """The pointer of an int32 tensor of this shape with unit stride in its last dimension."""
    if not (t.dtype is torch.int32 and t.shape == shape and t.get_device() == index and index >= 0
            and (t.stride()[-1] == 1 or shape[-1] <= 1)):
        _gpu(name, t, index)
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
        if t.stride(-1) != 1 and shape[-1] > 1:
            raise ValueError(f"{name} must have unit stride in its last dimension")
    return t.data_ptr()


def _table(name: str, t: torch.Tensor, index: int) -> tuple:
    """(rows, width, pointer, row stride) of a page table."""
    shape = t.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{name} must be [rows, pages] with at least one page, got {list(shape)}")
    p = _ints(name, t, shape, index)
    rows, width = shape
    ld = t.stride()[0] if rows > 1 else width
    if ld < width:
        raise ValueError(f"{name} must not have overlapping rows")
    return rows, width, p, ld


def _check_cache(k_pages, v_pages, index: int) -> None:
    """Raises what is wrong with the pools."""
    _gpu("k_pages", k_pages, index)
    _gpu("v_pages", v_pages, index)
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
        raise ValueError("k_pages and v_pages must both be [pages, HKV, page_size, D] of one dtype")
    if k_pages.dtype not in _KV:
        raise TypeError(f"pages must be bfloat16 or float8_e4m3fn, got {k_pages.dtype}")


def _scale(name: str, t, HKV: int, index: int) -> int:
    if t is None:
        raise ValueError("an e4m3 cache comes with k_scale and v_scale")
    _gpu(name, t, index)
    if t.dtype != torch.float32 or t.shape != (HKV,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 [{HKV}] tensor")
    return t.data_ptr()


def _cache(T: int, HQ: int, k_pages, v_pages, k_scale, v_scale, block_table, kv_lens, q_starts, index: int) -> tuple:
    """The fields of bz_paged_kv without the prefixes', checked."""
    # one expression for what is nearly always so; what it is not is found out afterwards
    shape, dtype, tshape = k_pages.shape, k_pages.dtype, block_table.shape
    if not (dtype in _KV and k_pages.get_device() == index and v_pages.get_device() == index and index >= 0
            and len(shape) == 4 and v_pages.shape == shape and v_pages.dtype is dtype):
        _check_cache(k_pages, v_pages, index)
    pages, HKV, ps, D = shape
    if dtype is not torch.bfloat16:
        ks, vs = _scale("k_scale", k_scale, HKV, index), _scale("v_scale", v_scale, HKV, index)
    elif k_scale is None and v_scale is None:
        ks = vs = 0
    else:
        raise ValueError("a bf16 cache has no scales")
    if (len(tshape) == 2 and kv_lens.dtype is block_table.dtype is torch.int32 and kv_lens.shape == tshape[:1]
            and kv_lens.get_device() == block_table.get_device() == index and kv_lens.stride()[0] == 1
            and (ts := block_table.stride())[1] == 1 and 1 <= tshape[1] <= ts[0]):
        B, width = tshape
        ld, table, lens = ts[0], block_table.data_ptr(), kv_lens.data_ptr()
    else:
        B, width, table, ld = _table("block_table", block_table, index)
        lens = _ints("kv_lens", kv_lens, (B,), index)
    if q_starts is not None:
        starts = _ints("q_starts", q_starts, (B + 1,), index)
    elif T == B:
        starts = 0
    else:
        raise ValueError(f"{T} rows for {B} sequences: q_starts says which are whose")
    k0, k1, k2, k3 = k_pages.stride()
    v0, v1, v2, v3 = v_pages.stride()
    if k3 != 1 or v3 != 1:
        raise ValueError("a position's D elements must be contiguous")
    # (strides of dimensions of size 1 are not used and count as D)
    if pages == 1:
        k0 = v0 = D
    if HKV == 1:
        k1 = v1 = D
    return ((_lib.ABI_VERSION, T, B, HQ, HKV, D, _KV[dtype], ps, pages, width),
            (k_pages.data_ptr(), v_pages.data_ptr(), k0, k1, k2, v0, v1, v2, ks, vs, table, ld, lens, starts))


_NO_PREFIX = (0, 0), (0, 0, 0, 0)


def _prefixes(table, lens, seqs, B: int, index: int) -> tuple:
    if table.dim() == 1:
        table = table.unsqueeze(0)
    groups, width, p, ld = _table("prefix_table", table, index)
    if groups < 1:
        raise ValueError("prefix_table needs at least one prefix")
    n = _ints("prefix_lens", lens, (groups,), index)
    if seqs is not None:
        at = _ints("prefix_seqs", seqs, (groups + 1,), index)
    elif groups == 1:
        at = 0
    else:
        raise ValueError("prefix_seqs says which sequences begin with which prefix")
    return (groups, width), (p, ld, n, at)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(sizes: tuple) -> int:
    d = _lib.paged_kv(*sizes, *(0,) * 18)
    return int(_lib.lib().bz_paged_attn_workspace(d))


def _heads(name: str, t: torch.Tensor) -> torch.Tensor:
    """[T, HQ, D] bf16 whose rows are contiguous, begin at multiples of 16 bytes and do not overlap."""
    shape = t.shape
    if len(shape) != 3 or t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be a bf16 [rows, HQ, D] tensor")
    a, b, c = t.stride()
    T, HQ, D = shape
    if t.data_ptr() % 16 or (c != 1 and D > 1) or (b != D and HQ > 1) or (T > 1 and (a % 8 or a < HQ * D)):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _result(name: str, t: torch.Tensor, shape: tuple, index: int, x: torch.Tensor) -> torch.Tensor:
    """A caller's output, checked, apart from the input x."""
    _gpu(name, t, index)
    inner = 1
    for n, s in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if n > 1 and s != inner:
            raise ValueError(f"{name} must have contiguous rows")
        inner *= n
    if t.dtype != torch.bfloat16 or t.shape != shape:
        raise ValueError(f"{name} must be a bf16 {list(shape)} tensor")
    if t.data_ptr() % 16 or (t.shape[0] > 1 and (t.stride(0) % 8 or t.stride(0) < inner)):
        raise ValueError(f"{name} needs rows at multiples of 16 bytes that do not overlap")
    if t.numel() and x.numel():
        end = t.data_ptr() + 2 * ((t.shape[0] - 1) * t.stride(0) + inner)
        if x.data_ptr() < end and t.data_ptr() < x.data_ptr() + 2 * ((x.shape[0] - 1) * x.stride(0) + x[0].numel()):
            raise ValueError(f"{name} must not overlap the input")
    return t


def _norm(name: str, w: torch.Tensor, D: int, index: int) -> torch.Tensor:
    """Norm weights as an aligned bf16 [D]."""
    if w.get_device() != index:
        _gpu(name, w, index)
    if w.numel() != D:
        raise ValueError(f"{name} must have {D} elements")
    if w.dtype != torch.bfloat16 or not w.is_contiguous() or w.data_ptr() % 16:
        w = w.to(torch.bfloat16).clone(memory_format=torch.contiguous_format)
    return w


def _call(index: int, stream: int, f, *args) -> None:
    """f(*args, stream) with the tensors' device current."""
    if torch._C._cuda_getDevice() == index:
        rc = f(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = f(*args, stream)
    if rc:
        raise _lib.BzError(rc, f.__name__)


def paged_rope_cache(qkv, cos, sin, k_pages, v_pages, block_table, kv_lens, HQ: int, q_starts=None, *, positions=None,
                     q_norm_w=None, k_norm_w=None, eps: float = 1e-6, k_scale=None, v_scale=None,
                     q_out=None) -> torch.Tensor:
    """Per-head q/k RMSNorm and rotate-half RoPE of the rows' qkv (bf16
    [T, (HQ + 2 HKV) D], q heads, k heads, v heads); their keys and values into
    the pages (e4m3: value / scale, rounded once, saturated; by a scale of 0 that is
    NaN for a value of 0); q as bf16 [T, HQ, D] (returned).
    What qkv_rope_cache does for a static cache, for any number of rows of
    each sequence.

    cos, sin: bf16 or fp32 [P, D], the rotary table.  Row t uses row positions[t]
    (int64 [T]), or without positions its own position in the sequence's pages; behind
    a shared prefix pass positions.  A row outside the table is written to no page
    and its q is zero."""
    index = qkv.get_device()
    shape = qkv.shape
    if index < 0:
        _gpu("qkv", qkv, index)
    if len(shape) != 2 or qkv.dtype != torch.bfloat16:
        raise ValueError("qkv must be a bf16 [rows, (HQ + 2 HKV) D] tensor")
    T, width = shape
    sizes, refs = _cache(T, HQ, k_pages, v_pages, k_scale, v_scale, block_table, kv_lens, q_starts, index)
    HKV, D = sizes[4], sizes[5]
    if HQ < 1 or width != (HQ + 2 * HKV) * D:
        raise ValueError(f"qkv width {width} is not ({HQ} + 2 * {HKV}) heads of {D}")
    ld, inner = qkv.stride()
    if inner != 1 or qkv.data_ptr() % 16 or (T > 1 and (ld % 8 or ld < width)):
        qkv = qkv.clone(memory_format=torch.contiguous_format)
        ld = width
    if cos.dim() == 3 and cos.shape[0] == 1:
        cos, sin = cos[0], sin[0] if sin.dim() == 3 else sin
    shape, cs = cos.shape, _CS.get(cos.dtype)
    if not (cos.get_device() == index and sin.get_device() == index and len(shape) == 2 and sin.shape == shape
            and sin.dtype == cos.dtype and shape[1] == D and shape[0] > 0 and cs is not None):
        for name, t in (("cos", cos), ("sin", sin)):
            _gpu(name, t, index)
        if cos.dim() != 2 or shape != sin.shape or cos.dtype != sin.dtype or shape[1] != D or shape[0] < 1:
            raise ValueError(f"cos and sin must both be [positions, {D}] of one dtype")
        raise TypeError(f"cos and sin must be bfloat16 or float32, got {cos.dtype}")
    ld_cs, inner = cos.stride()
    if sin.stride() != (ld_cs, inner) or inner != 1 or (shape[0] > 1 and (ld_cs % 8 or ld_cs < D)) \
            or cos.data_ptr() % 16 or sin.data_ptr() % 16:
        cos, sin = (t.clone(memory_format=torch.contiguous_format) for t in (cos, sin))
        ld_cs = D
    at = 0
    if positions is not None:
        _gpu("positions", positions, index)
        if positions.dtype != torch.int64 or positions.shape != (T,) or not positions.is_contiguous():
            raise ValueError(f"positions must be a contiguous int64 [{T}] tensor")
        at = positions.data_ptr()
    qn = kn = None
    if q_norm_w is not None and k_norm_w is not None:
        qn, kn = _norm("q_norm_w", q_norm_w, D, index), _norm("k_norm_w", k_norm_w, D, index)
    elif q_norm_w is not None or k_norm_w is not None:
        raise ValueError("q_norm_w and k_norm_w come together")
    q = qkv.new_empty((T, HQ, D)) if q_out is None else _result("q_out", q_out, (T, HQ, D), index, qkv)
    if T == 0 or sizes[2] == 0:
        return q
    _call(index, torch._C._cuda_getCurrentRawStream(index), _lib.lib().bz_paged_rope_cache,
          _lib.paged_kv(*sizes, 0, 0, *refs, 0, 0, 0, 0), qkv.data_ptr(), ld if T > 1 else width,
          None if qn is None else qn.data_ptr(), None if kn is None else kn.data_ptr(), eps, cos.data_ptr(),
          sin.data_ptr(), cs, ld_cs if shape[0] > 1 else D, shape[0], at, q.data_ptr(), q.stride()[0] if T > 1 else HQ * D)
    return q


def _attention(q, k_pages, v_pages, block_table, kv_lens, q_starts, prefix, scale, k_scale, v_scale, out):
    index = q.get_device()
    if index < 0:
        _gpu("q", q, index)
    q = _heads("q", q)
    T, HQ, D = q.shape
    sizes, refs = _cache(T, HQ, k_pages, v_pages, k_scale, v_scale, block_table, kv_lens, q_starts, index)
    if D != sizes[5]:
        raise ValueError(f"q has heads of {D}, the pages of {sizes[5]}")
    psizes, prefs = _NO_PREFIX if prefix is None else _prefixes(*prefix, sizes[2], index)
    width = HQ * D
    if out is None:
        out, ld = q.new_empty((T, width)), width
    else:
        out = _result("out", out, (T, width), index, q)
        ld = out.stride()[0] if T > 1 else width
    if T == 0 or sizes[2] == 0:
        return out
    sizes += psizes
    n = _workspace_bytes(sizes)
    stream = torch._C._cuda_getCurrentRawStream(index)
    kv = _lib.paged_kv(*sizes, *refs, *prefs)
    lock = _LOCKS.get((index, stream))
    if lock is None:
        lock = _LOCKS.setdefault((index, stream), threading.RLock())
    with lock:
        ws = _lib.stream_workspace(_WS, (index,), n, q.device, stream, _WS_RETIRED)
        _call(index, stream, _lib.lib().bz_paged_attn, kv, q.data_ptr(), q.stride()[0] if T > 1 else width,
              D ** -0.5 if scale is None else scale, ws.data_ptr(), n, out.data_ptr(), ld)
    return out


def paged_attention(q, k_pages, v_pages, block_table, kv_lens, q_starts=None, *, scale: Optional[float] = None,
                    k_scale=None, v_scale=None, out=None) -> torch.Tensor:
    """softmax(scale q k^T) v of every row over its sequence's positions up to the
    row's own: q bf16 [T, HQ, D], rotated -> bf16 [T, HQ * D].  Query head h
    reads key/value head h // (HQ / HKV).  One row per sequence is a decode step,
    several are drafted tokens, a prompt or a chunk of one.  scale: D ** -0.5
    unless given, positive.  A row that attends nothing is zero; keys and values that
    a row does not attend have no part in it, whatever they hold."""
    return _attention(q, k_pages, v_pages, block_table, kv_lens, q_starts, None, scale, k_scale, v_scale, out)


def shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_lens, block_table, kv_lens, q_starts=None,
                            prefix_seqs=None, *, scale: Optional[float] = None, k_scale=None, v_scale=None,
                            out=None) -> torch.Tensor:
    """paged_attention for sequences that begin with a shared prefix: prefix g, of
    prefix_lens[g] positions (int32 [groups]) in the pages prefix_table[g] (int32
    [groups, W'], or [W'] for one), comes before the own positions of the
    sequences prefix_seqs[g] .. prefix_seqs[g + 1] - 1 (int32 [groups + 1]; None with one
    prefix: of all).  Every row attends its whole prefix, then its sequence's own
    positions as in paged_attention; kv_lens and block_table are about the own
    positions alone, and kv_lens may leave a row none of them.  The prefix's keys and
    values are read once for every 16 to 128 of its sequences' query rows of a key/value
    head, not once for each sequence."""
    return _attention(q, k_pages, v_pages, block_table, kv_lens, q_starts, (prefix_table, prefix_lens, prefix_seqs),
                      scale, k_scale, v_scale, out)
