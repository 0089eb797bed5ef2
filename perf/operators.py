"""Operators over a paged key/value cache, as measurable cases.

A speech server holds the keys and values of its requests in pages of a pool.  Three operators work on it:

``append``   the new tokens' q/k norm and rotary embedding; their keys and values into the pages (bf16, or e4m3 with a
             scale per key/value head), their rotated queries to a tensor
``attend``   attention of each sequence's newest rows (one token, a few drafted ones, a prompt or a chunk of one) over
             its pages, causal from the end
``prefix``   the same for batches whose sequences begin with a shared prompt, stored once per group of sequences

The served model pairs a backbone of 16 query and 8 key/value heads of 128 with a depth decoder of 8 and 2 heads of 128;
16 and 4 heads of 256 is the wider geometry that the benchmark measures.  Lengths, pages and values of a case come from
the case; tokens, page order and contents from the seed.
"""

import functools
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 1e6
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def listed():
    return [
        # the step of one request with guidance (a conditional and an unconditional row), some 600 positions in
        {"name": "append_step_b2", "kind": "append", "HQ": 16, "HKV": 8, "D": 128, "ps": 16, "kv": "bf16", "B": 2,
         "n_lo": 1, "n_hi": 1, "c_lo": 610, "c_hi": 610},
        # the prompts of seven requests, of different lengths, admitted at once
        {"name": "append_prompts_b7", "kind": "append", "HQ": 16, "HKV": 4, "D": 256, "ps": 64, "kv": "bf16", "B": 7,
         "n_lo": 33, "n_hi": 611, "c_lo": 0, "c_hi": 0},
        # a chunk of a long reference recording's prompt, cache in 8 bits
        {"name": "append_chunk_e4m3", "kind": "append", "HQ": 16, "HKV": 8, "D": 128, "ps": 32, "kv": "e4m3", "B": 1,
         "n_lo": 8191, "n_hi": 8191, "c_lo": 4096, "c_hi": 4096},
        # the attention of that one request's step: the smallest call there is
        {"name": "decode_b2", "kind": "attend", "HQ": 16, "HKV": 8, "D": 128, "ps": 16, "kv": "bf16", "B": 2,
         "n_lo": 1, "n_hi": 1, "c_lo": 610, "c_hi": 610},
        # a full server: 48 rows, anything from a fresh request to the end of a long one
        {"name": "decode_b48", "kind": "attend", "HQ": 16, "HKV": 8, "D": 128, "ps": 64, "kv": "bf16", "B": 48,
         "n_lo": 1, "n_hi": 1, "c_lo": 40, "c_hi": 4095},
        # few rows over very long contexts, cache in 8 bits
        {"name": "decode_long_e4m3", "kind": "attend", "HQ": 16, "HKV": 4, "D": 256, "ps": 128, "kv": "e4m3", "B": 4,
         "n_lo": 1, "n_hi": 1, "c_lo": 30011, "c_hi": 65535},
        # verification of five drafted tokens for each of 16 rows
        {"name": "verify_b16_n5", "kind": "attend", "HQ": 8, "HKV": 2, "D": 128, "ps": 16, "kv": "bf16", "B": 16,
         "n_lo": 5, "n_hi": 5, "c_lo": 97, "c_hi": 2043},
        # the prompt of one request, an odd number of positions
        {"name": "prompt_2011", "kind": "attend", "HQ": 16, "HKV": 8, "D": 128, "ps": 16, "kv": "bf16", "B": 1,
         "n_lo": 2011, "n_hi": 2011, "c_lo": 0, "c_hi": 0},
        # chunks of three long prompts, of different lengths, over what is already there
        {"name": "chunks_b3", "kind": "attend", "HQ": 16, "HKV": 4, "D": 256, "ps": 16, "kv": "bf16", "B": 3,
         "n_lo": 301, "n_hi": 1024, "c_lo": 1000, "c_hi": 8000},
        # four requests of one voice with guidance: the voice's prompt for the conditional rows, a short one for the others
        {"name": "prefix_voice_b8", "kind": "prefix", "HQ": 16, "HKV": 8, "D": 128, "ps": 16, "kv": "bf16", "B": 8,
         "n_lo": 1, "n_hi": 1, "c_lo": 3, "c_hi": 200, "groups": 2, "p_lo": 41, "p_hi": 301},
        # 64 requests of one voice with a long reference recording
        {"name": "prefix_b64", "kind": "prefix", "HQ": 16, "HKV": 8, "D": 128, "ps": 64, "kv": "bf16", "B": 64,
         "n_lo": 1, "n_hi": 1, "c_lo": 1, "c_hi": 511, "groups": 1, "p_lo": 6007, "p_hi": 6007},
        # three long prompts in 8 bits, eight requests each, two tokens a step
        {"name": "prefix_b24_e4m3", "kind": "prefix", "HQ": 16, "HKV": 4, "D": 256, "ps": 128, "kv": "e4m3", "B": 24,
         "n_lo": 2, "n_hi": 2, "c_lo": 100, "c_hi": 1500, "groups": 3, "p_lo": 9001, "p_hi": 16383},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "prefix", "prefix"])
    hq, hkv, d = rng.choice([(16, 8, 128), (16, 8, 128), (8, 2, 128), (16, 4, 256), (6, 2, 64), (9, 3, 128), (16, 1, 64),
                             (4, 4, 128)])
    case = {"kind": kind, "HQ": hq, "HKV": hkv, "D": d, "ps": rng.choice([16, 16, 32, 64, 128, 256]),
            "kv": rng.choice(["bf16", "bf16", "e4m3"])}
    if kind == "append":
        if rng.random() < 0.5:  # steps
            case |= {"B": _spread(rng, 1, 128), "n_lo": 1, "n_hi": rng.choice([1, 1, 5]), "c_lo": 0,
                     "c_hi": _spread(rng, 16, 2048)}
        else:  # prompts and chunks of them
            b = _spread(rng, 1, 8)
            n = _spread(rng, 17, 8191 // b)
            case |= {"B": b, "n_lo": _spread(rng, 1, n), "n_hi": n, "c_lo": 0, "c_hi": rng.choice([0, 511, 2048])}
        return case
    form = rng.choice(["step", "step", "few", "prompt"]) if kind == "attend" else "step"
    if form == "prompt":
        b = _spread(rng, 1, 4)
        n = _spread(rng, 33, 2048 // b)
        case |= {"B": b, "n_lo": _spread(rng, 1, n), "n_hi": n, "c_lo": 0, "c_hi": rng.choice([0, 0, 777, 4000])}
    else:
        b = _spread(rng, 1, 64)
        top = 4096 if kind == "attend" else 1024
        c = _spread(rng, 8, max(top, min(32768, 65536 // b)) if kind == "attend" else top)
        n = 1 if form == "step" and kind == "attend" else rng.choice([1, 1, 2, 5]) if kind == "prefix" else rng.randint(2, 9)
        case |= {"B": b, "n_lo": n, "n_hi": n, "c_lo": _spread(rng, 1, c), "c_hi": c}
    if kind == "prefix":
        case |= {"groups": rng.choice([1, 1, 2, 3]) if case["B"] > 3 else 1, "p_hi": _spread(rng, 40, 16384)}
        case["p_lo"] = _spread(rng, 17, case["p_hi"])
    return case


def _lengths(count, lo, hi):
    """``count`` lengths from lo to hi in no order, the first the longest."""
    return [lo + int(((i * 0.6180339887498949 + 0.999) % 1.0) * (hi - lo + 1)) for i in range(count)]


def _shape(case):
    """New rows and own length (with them) of each sequence, length of each prefix, sequences of each group."""
    b, groups = case["B"], case.get("groups", 0)
    n = _lengths(b, case["n_lo"], case["n_hi"])
    kv = [c + m for c, m in zip(_lengths(b, case["c_lo"], case["c_hi"]), n)]
    p = _lengths(groups, case["p_lo"], case["p_hi"]) if groups else []
    seqs = [b * g // groups for g in range(groups + 1)] if groups else []
    return n, kv, p, seqs


def work(case):
    n, kv, p, seqs = _shape(case)
    hq, hkv, d, es = case["HQ"], case["HKV"], case["D"], 2 if case["kv"] == "bf16" else 1
    rows = sum(n)
    if case["kind"] == "append":
        return {"bytes": rows * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + 2 * hkv * d * es + 2 * d * 4),
                "flops": rows * (hq + hkv) * d * 7}
    pairs = sum(m * (k - m) + m * (m + 1) // 2 for m, k in zip(n, kv))
    for g, length in enumerate(p):
        pairs += length * sum(n[seqs[g]:seqs[g + 1]])
    return {"bytes": rows * hq * d * 4 + (sum(kv) + sum(p)) * hkv * d * 2 * es, "flops": 4 * d * hq * pairs}


# ---- what a program has in hand before the call ----------------------------------------------------


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(n):
    at = [0]
    for m in n:
        at.append(at[-1] + m)
    return at


def _pool(g, pages, hkv, ps, d, kv, spread):
    """Keys (or values) of a whole pool: every position holds something, as after an hour of serving."""
    t = torch.randn(pages, hkv, ps, d, device=DEV, generator=g) * spread
    if kv == "bf16":
        return t.to(BF16), None
    scale = torch.linspace(0.75, 1.25, hkv, device=DEV) * spread * 5 / 448
    return (t / scale[:, None, None]).clamp(-448, 448).to(E4M3), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n, kv, p, seqs = _shape(case)
    hq, hkv, d, ps = case["HQ"], case["HKV"], case["D"], case["ps"]
    rows, starts = sum(n), _starts(n)
    width = -(-max(kv) // ps)
    p_width = -(-max(p) // ps) if p else 0
    pages = len(kv) * width + len(p) * p_width + 3
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)  # pages of a request lie anywhere in the pool
    s = {"case": case, "kv_lens": _i32(kv), "table": order[: len(kv) * width].view(len(kv), width).contiguous(),
         "starts": None if n == [1] * len(n) else _i32(starts)}
    s["k"], s["k_scale"] = _pool(g, pages, hkv, ps, d, case["kv"], 1.5)
    s["v"], s["v_scale"] = _pool(g, pages, hkv, ps, d, case["kv"], 1.0)
    if case["kind"] == "append":
        top = max(kv)
        inv = THETA ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
        angle = (torch.arange(top, device=DEV, dtype=torch.float64)[:, None] * inv).repeat(1, 2)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()  # the rotary table of the positions served
        s["qkv"] = torch.randn(rows, (hq + 2 * hkv) * d, device=DEV, generator=g).to(BF16)
        s["qn"], s["kn"] = ((1 + 0.1 * torch.randn(d, device=DEV, generator=g)).to(BF16) for _ in range(2))
        return s
    s["q"] = (torch.randn(rows, hq, d, device=DEV, generator=g) * 1.5).to(BF16)
    if p:
        s["p_table"] = order[len(kv) * width: len(kv) * width + len(p) * p_width].view(len(p), p_width).contiguous()
        s["p_lens"], s["p_seqs"] = _i32(p), _i32(seqs)
    return s


# ---- one pass ---------------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _paged():
    sys.path.insert(0, os.path.join(os.getcwd(), "breeze-tts-2_amd"))
    from breeze_amd import paged

    return paged


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return _plain_append(s) if kind == "append" else _plain_attention(s)
    if kind == "append":
        q = _paged().paged_rope_cache(s["qkv"], s["cos"], s["sin"], s["k"], s["v"], s["table"], s["kv_lens"],
                                      s["case"]["HQ"], s["starts"], q_norm_w=s["qn"], k_norm_w=s["kn"], eps=EPS,
                                      k_scale=s["k_scale"], v_scale=s["v_scale"])
        return q, s["k"], s["v"]
    if kind == "attend":
        return _paged().paged_attention(s["q"], s["k"], s["v"], s["table"], s["kv_lens"], s["starts"],
                                        k_scale=s["k_scale"], v_scale=s["v_scale"])
    return _paged().shared_prefix_attention(s["q"], s["k"], s["v"], s["p_table"], s["p_lens"], s["table"], s["kv_lens"],
                                            s["starts"], s["p_seqs"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _rows(s, rows):
    """Sequence, place in it and own position of each row; rows of each sequence."""
    b = s["kv_lens"].numel()
    starts = torch.arange(b + 1, device=DEV) if s["starts"] is None else s["starts"].long()
    t = torch.arange(rows, device=DEV)
    seq = torch.bucketize(t, starts[1:], right=True)
    place = t - starts[seq]
    n = starts[1:] - starts[:-1]
    return seq, place, s["kv_lens"].long()[seq] - n[seq] + place, n


def _norm_rope(x, w, cos, sin):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    h = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat([-x[..., h:], x[..., :h]], -1) * sin[:, None]


def _put(pages, scale, page, at, x):
    if scale is None:
        pages[page, :, at] = x.to(pages.dtype)
    else:
        code = (x.float() / scale[:, None]).clamp(-448, 448).to(E4M3)
        pages.view(torch.uint8)[page, :, at] = code.view(torch.uint8)


def _plain_append(s):
    hq, hkv, d, ps = (s["case"][k] for k in ("HQ", "HKV", "D", "ps"))
    x = s["qkv"].view(-1, hq + 2 * hkv, d)
    seq, _, pos, _ = _rows(s, x.shape[0])
    cos, sin = s["cos"][pos], s["sin"][pos]
    page, at = s["table"].long()[seq, pos // ps], pos % ps
    _put(s["k"], s["k_scale"], page, at, _norm_rope(x[:, hq:hq + hkv], s["kn"], cos, sin))
    _put(s["v"], s["v_scale"], page, at, x[:, hq + hkv:])
    return _norm_rope(x[:, :hq], s["qn"], cos, sin).to(BF16), s["k"], s["v"]


def _take(pages, scale, page, at):
    """[B, L] places -> fp32 [B, HKV, L, D]."""
    if scale is None:
        x = pages[page, :, at].float()
    else:
        x = pages.view(torch.uint8)[page, :, at].view(E4M3).float() * scale[:, None]
    return x.permute(0, 2, 1, 3).contiguous()


def _plain_attention(s):
    hq, hkv, d, ps = (s["case"][k] for k in ("HQ", "HKV", "D", "ps"))
    rows, lens = s["q"].shape[0], s["kv_lens"].long()
    seq, place, pos, n = _rows(s, rows)
    b, top_n, group = lens.numel(), s["case"]["n_hi"], hq // hkv
    # where key j of a sequence lies: the first prefix_len of them in its group's pages, then its own
    width = s["table"].shape[1] * ps
    if "p_lens" in s:
        width += s["p_table"].shape[1] * ps
        of = torch.bucketize(torch.arange(b, device=DEV), s["p_seqs"].long()[1:], right=True)
        before = s["p_lens"].long()[of][:, None]
    else:
        before = torch.zeros(b, 1, dtype=torch.long, device=DEV)
    j = torch.arange(width, device=DEV)[None].expand(b, width)
    mine = (j - before).clamp(0, s["table"].shape[1] * ps - 1)
    page, at = s["table"].long().gather(1, mine // ps), mine % ps
    if "p_lens" in s:
        first = j.clamp(max=s["p_table"].shape[1] * ps - 1)
        page = torch.where(j < before, s["p_table"].long()[of].gather(1, first // ps), page)
        at = torch.where(j < before, first % ps, at)
    k, v = _take(s["k"], s["k_scale"], page, at), _take(s["v"], s["v_scale"], page, at)
    q = torch.zeros(b, top_n, hkv, group, d, device=DEV)
    q[seq, place] = s["q"].view(rows, hkv, group, d).float()
    q = q.permute(0, 2, 1, 3, 4).reshape(b, hkv, top_n * group, d)
    w = torch.matmul(q, k.transpose(2, 3).contiguous()).view(b, hkv, top_n, group, width) * d ** -0.5
    # row i of a sequence is its own position lens - n + i, and sees what is not behind it
    last = before + (lens - n)[:, None] + torch.arange(top_n, device=DEV)
    w = w.masked_fill((j[:, None] > last[..., None])[:, None, :, None], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(b, hkv, top_n * group, width), v).view(b, hkv, top_n, group, d)
    return out.permute(0, 2, 1, 3, 4)[seq, place].reshape(rows, hq * d).to(BF16)


# ---- the definition, in 64 bits, one sequence after the other ----------------------------------------


def _exact_append(s):
    case = s["case"]
    hq, hkv, d, ps = (case[k] for k in ("HQ", "HKV", "D", "ps"))
    n, kv, _, _ = _shape(case)
    k = s["k"].double() if s["k_scale"] is None else s["k"].float().double()
    v = s["v"].double() if s["v_scale"] is None else s["v"].float().double()
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    q = torch.empty(x.shape[0], hq, d, dtype=torch.float64, device=DEV)

    def turned(y, w, c, z):
        y = y / (y.square().sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        a, b = y[..., : d // 2], y[..., d // 2:]
        c, z = c[:, None], z[:, None]
        return torch.cat([a * c[..., : d // 2] - b * z[..., : d // 2], b * c[..., d // 2:] + a * z[..., d // 2:]], -1)

    row = 0
    for b, (m, length) in enumerate(zip(n, kv)):
        for lo in range(0, m, 2048):
            part = slice(row + lo, row + min(m, lo + 2048))
            pos = torch.arange(length - m + lo, length - m + min(m, lo + 2048), device=DEV)
            cos, sin = s["cos"][pos].double(), s["sin"][pos].double()
            q[part] = turned(x[part, :hq], s["qn"], cos, sin)
            page, at = s["table"][b].long()[pos // ps], pos % ps
            new_k, new_v = turned(x[part, hq:hq + hkv], s["kn"], cos, sin), x[part, hq + hkv:]
            if s["k_scale"] is not None:
                new_k = (new_k / s["k_scale"].double()[:, None]).clamp(-448, 448)
                new_v = (new_v / s["v_scale"].double()[:, None]).clamp(-448, 448)
            k[page, :, at] = new_k
            v[page, :, at] = new_v
        row += m
    return q, k, v


def _exact_attention(s):
    case = s["case"]
    hq, hkv, d, ps = (case[k] for k in ("HQ", "HKV", "D", "ps"))
    n, kv, p, seqs = _shape(case)
    out = torch.empty(sum(n), hq, d, dtype=torch.float64, device=DEV)

    def rows_of(table, length):
        pages = table[: -(-length // ps)].long()
        for pool, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
            x = (pool if scale is None else pool.view(torch.uint8))[pages]
            x = x.double() if scale is None else x.view(E4M3).double() * scale.double()[:, None, None]
            yield x.transpose(0, 1).reshape(hkv, -1, d)[:, :length]

    row = 0
    for b, (m, length) in enumerate(zip(n, kv)):
        k, v = rows_of(s["table"][b], length)
        before = 0
        if p:
            g = max(i for i in range(len(p)) if seqs[i] <= b)
            before = p[g]
            first_k, first_v = rows_of(s["p_table"][g], before)
            k, v = torch.cat([first_k, k], 1), torch.cat([first_v, v], 1)
        j = torch.arange(before + length, device=DEV)
        for lo in range(0, m, 256):
            hi = min(m, lo + 256)
            last = torch.arange(before + length - m + lo, before + length - m + hi, device=DEV)
            for h in range(hq):
                score = s["q"][row + lo:row + hi, h].double() @ k[h * hkv // hq].T / math.sqrt(d)
                score = score.masked_fill(j > last[:, None], -math.inf)
                out[row + lo:row + hi, h] = torch.softmax(score, -1) @ v[h * hkv // hq]
        row += m
    return out.view(sum(n), hq * d)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attention(s)
