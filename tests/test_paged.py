"""The operators over a paged cache without a GPU: the oracle against torch, the
wrappers' refusals, and the C ABI's answers to bad arguments before anything touches
a device."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
import threading
import time
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import bz_paged_oracle as P
from tests._paged import BF16, E4M3, Cache, ints, starts_of
from tests._paged_parts import KEYS, PROB, VALUE, half_step, parts_bound

from breeze_amd import _lib, paged

ROOT = Path(__file__).resolve().parents[1]


def test_oracle_is_softmax_attention():
    """Against torch's attention in 64 bits over the gathered sequence."""
    rng = np.random.default_rng(0)
    cache = Cache(rng, 30, 2, 16, 64, dev="cpu")
    table, ptable = cache.table(3, 4), cache.table(1, 2)
    lens, n, plen = [50, 7, 33], [3, 7, 1], 20
    starts = starts_of(n)
    q = rng.standard_normal((int(starts[-1]), 6, 64))
    k, v = cache.values("k"), cache.values("v")
    got, weight, size = P.attention(q, k, v, table.numpy(), lens, starts, None, (ptable.numpy(), [plen], None))
    for b in range(3):
        seq = lambda pool: torch.from_numpy(np.concatenate([  # noqa: E731
            pool[ptable[0].numpy()].transpose(1, 0, 2, 3).reshape(2, -1, 64)[:, :plen],
            pool[table[b].numpy()].transpose(1, 0, 2, 3).reshape(2, -1, 64)[:, :lens[b]]], 1)).repeat_interleave(3, 0)
        rows = torch.from_numpy(q[starts[b]:starts[b + 1]]).transpose(0, 1)
        allow = torch.ones(n[b], plen + lens[b]).tril(plen + lens[b] - n[b]).bool()
        want = torch.nn.functional.scaled_dot_product_attention(rows, seq(k), seq(v), attn_mask=allow)
        np.testing.assert_allclose(got[starts[b]:starts[b + 1]], want.transpose(0, 1).numpy(), rtol=1e-10, atol=1e-12)


def test_oracle_rows_and_slots():
    assert P.rows_of(6, 2, [5, 1], [1, 3, 5]) == [(1, 0, 3), (2, 0, 4), (3, 1, -1), (4, 1, 0)]
    assert P.rows_of(2, 2, [5, 0], None) == [(0, 0, 4), (1, 1, -1)]
    assert P.slot([3, -1], 5, 16, 4) == (3, 5) and P.slot([3, -1], 17, 16, 4) is None
    assert P.slot([3, 4], 17, 16, 4) is None and P.slot([3], 16, 16, 4) is None and P.slot([3], -1, 16, 4) is None


def test_oracle_rope_is_a_rotation():
    rng = np.random.default_rng(1)
    x, th = rng.standard_normal((5, 64)), rng.uniform(-3, 3, 32)
    cos, sin = (np.tile(f(th), 2) for f in (np.cos, np.sin))
    y, _ = P.norm_rope(x, None, 0.0, cos, sin)
    z = (x[:, :32] + 1j * x[:, 32:]) * np.exp(1j * th)
    np.testing.assert_allclose(y, np.concatenate([z.real, z.imag], -1), rtol=1e-12)
    y, _ = P.norm_rope(x, np.ones(64), 0.0, cos, sin)
    np.testing.assert_allclose((y * y).mean(-1), 1.0, rtol=1e-12)


# ---- the wrappers ---------------------------------------------------------------------------------


@pytest.fixture
def no_gpu(monkeypatch):
    """The wrappers' checks on CPU tensors: the device check passes, and a call that
    reaches the library fails the test."""
    monkeypatch.setattr(paged, "_gpu", lambda *a: None)

    def reached(*a):
        raise AssertionError("reached the library")

    monkeypatch.setattr(paged, "_call", reached)
    monkeypatch.setattr(paged, "_workspace_bytes", reached)


def _args(kv="bf16", **kw):
    rng = np.random.default_rng(2)
    c = Cache(rng, 8, 2, 16, 64, kv, dev="cpu")
    a = {"q": torch.zeros(3, 4, 64, dtype=BF16), "k_pages": c.k, "v_pages": c.v, "block_table": ints([[0], [1], [2]], "cpu"),
         "kv_lens": ints([1, 2, 3], "cpu"), "k_scale": c.k_scale, "v_scale": c.v_scale}
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error", [
    ({"q": torch.zeros(3, 256, dtype=BF16)}, ValueError),
    ({"q": torch.zeros(3, 4, 64)}, ValueError),
    ({"q": torch.zeros(3, 4, 128, dtype=BF16)}, ValueError),
    ({"q": torch.zeros(4, 4, 64, dtype=BF16)}, ValueError),                    # rows without q_starts
    ({"k_pages": torch.zeros(8, 2, 16, 64)}, ValueError),                      # not v_pages' dtype
    ({"k_pages": torch.zeros(8, 2, 16, 32, dtype=BF16)}, ValueError),
    ({"k_pages": torch.zeros(8, 2, 16, dtype=BF16), "v_pages": torch.zeros(8, 2, 16, dtype=BF16)}, ValueError),
    ({"k_pages": torch.zeros(8, 2, 16, 64), "v_pages": torch.zeros(8, 2, 16, 64)}, TypeError),
    ({"k_pages": torch.zeros(8, 2, 64, 16, dtype=BF16).transpose(2, 3)}, ValueError),
    ({"k_scale": torch.ones(2)}, ValueError),                                  # a bf16 cache has no scales
    ({"block_table": torch.zeros(3, 1, dtype=torch.int64)}, TypeError),
    ({"block_table": torch.zeros(3, dtype=torch.int32)}, ValueError),
    ({"block_table": torch.zeros(3, 0, dtype=torch.int32)}, ValueError),
    ({"block_table": torch.zeros(2, 3, dtype=torch.int32).t()[:, ::2]}, None),
    ({"block_table": torch.zeros(1, 1, dtype=torch.int32).expand(3, 1)}, ValueError),
    ({"block_table": torch.zeros(2, 3, dtype=torch.int32).t()}, ValueError),
    ({"kv_lens": torch.zeros(2, dtype=torch.int32)}, ValueError),
    ({"kv_lens": torch.zeros(3, dtype=torch.int64)}, TypeError),
    ({"kv_lens": torch.zeros(6, dtype=torch.int32)[::2]}, ValueError),
    ({"q_starts": torch.zeros(3, dtype=torch.int32)}, ValueError),
    ({"out": torch.zeros(3, 256)}, ValueError),
    ({"out": torch.zeros(3, 128, dtype=BF16)}, ValueError),
    ({"out": torch.zeros(3, 260, dtype=BF16)[:, :256]}, ValueError),
    ({"out": torch.zeros(3, 264, dtype=BF16)[:, 4:260]}, ValueError),
    ({"out": torch.zeros(256, dtype=BF16).expand(3, 256)}, ValueError),
    ({"out": torch.zeros(3, 512, dtype=BF16)[:, ::2]}, ValueError),
])
def test_attention_refuses(no_gpu, kw, error):
    if error is None:
        with pytest.raises(AssertionError, match="reached"):
            paged.paged_attention(**_args(**kw))
        return
    with pytest.raises(error):
        paged.paged_attention(**_args(**kw))


@pytest.mark.parametrize("kw", [{"k_scale": None}, {"v_scale": None}, {"k_scale": torch.ones(3)},
                                {"k_scale": torch.ones(2, dtype=torch.float64)}, {"v_scale": torch.ones(4)[::2]}])
def test_e4m3_needs_its_scales(no_gpu, kw):
    with pytest.raises(ValueError):
        paged.paged_attention(**_args("e4m3", **kw))


def test_out_must_not_be_the_input(no_gpu):
    q = torch.zeros(3, 4, 64, dtype=BF16)
    with pytest.raises(ValueError, match="overlap"):
        paged.paged_attention(**_args(q=q, out=q.view(3, 256)))
    wide = torch.zeros(4, 256, dtype=BF16)
    with pytest.raises(ValueError, match="overlap"):
        paged.paged_attention(**_args(q=wide[:3].view(3, 4, 64), out=wide[1:]))


@pytest.mark.parametrize("kw,error", [
    ({"prefix_table": torch.zeros(2, 1, dtype=torch.int32)}, ValueError),      # two prefixes, one length
    ({"prefix_lens": torch.zeros(1, dtype=torch.int64)}, TypeError),
    ({"prefix_table": torch.zeros(2, 1, dtype=torch.int32), "prefix_lens": torch.zeros(2, dtype=torch.int32)}, ValueError),
    ({"prefix_table": torch.zeros(0, 1, dtype=torch.int32), "prefix_lens": torch.zeros(0, dtype=torch.int32)}, ValueError),
    ({"prefix_seqs": torch.zeros(3, dtype=torch.int32)}, ValueError),
])
def test_prefix_refuses(no_gpu, kw, error):
    a = _args(prefix_table=torch.zeros(1, dtype=torch.int32), prefix_lens=torch.zeros(1, dtype=torch.int32))
    a.update(kw)
    with pytest.raises(error):
        paged.shared_prefix_attention(**a)


def _rope_args(**kw):
    a = _args()
    a = {k: a[k] for k in ("k_pages", "v_pages", "block_table", "kv_lens")}
    a |= {"qkv": torch.zeros(3, 8 * 64, dtype=BF16), "cos": torch.zeros(5, 64), "sin": torch.zeros(5, 64), "HQ": 4}
    return a | kw


@pytest.mark.parametrize("kw,error", [
    ({"qkv": torch.zeros(3, 8 * 64)}, ValueError),
    ({"qkv": torch.zeros(3, 7 * 64, dtype=BF16)}, ValueError),
    ({"HQ": 5}, ValueError),
    ({"HQ": 0, "qkv": torch.zeros(3, 4 * 64, dtype=BF16)}, ValueError),
    ({"cos": torch.zeros(5, 32)}, ValueError),
    ({"cos": torch.zeros(4, 64)}, ValueError),
    ({"cos": torch.zeros(5, 64, dtype=BF16)}, ValueError),
    ({"cos": torch.zeros(3, 1, 64), "sin": torch.zeros(3, 1, 64)}, ValueError),
    ({"cos": torch.zeros(0, 64), "sin": torch.zeros(0, 64)}, ValueError),
    ({"cos": torch.zeros(5, 64).half(), "sin": torch.zeros(5, 64).half()}, TypeError),
    ({"positions": torch.zeros(3, dtype=torch.int32)}, ValueError),
    ({"positions": torch.zeros(2, dtype=torch.int64)}, ValueError),
    ({"q_norm_w": torch.ones(64)}, ValueError),
    ({"q_norm_w": torch.ones(64), "k_norm_w": torch.ones(32)}, ValueError),
    ({"q_out": torch.zeros(3, 4, 64)}, ValueError),
    ({"q_out": torch.zeros(3, 4, 128, dtype=BF16)[:, :, ::2]}, ValueError),
])
def test_append_refuses(no_gpu, kw, error):
    with pytest.raises(error):
        paged.paged_rope_cache(**_rope_args(**kw))


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        paged.paged_attention(**_args())
    with pytest.raises(RuntimeError, match="GPU"):
        paged.paged_rope_cache(**_rope_args())
    with pytest.raises(RuntimeError, match="GPU"):
        paged.shared_prefix_attention(**_args(prefix_table=torch.zeros(1, dtype=torch.int32),
                                              prefix_lens=torch.zeros(1, dtype=torch.int32)))


# ---- the C ABI ------------------------------------------------------------------------------------


def test_descriptor_layout_matches_c(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc not available")
    fields = [f for f, _ in _lib.PagedKv._fields_]
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "bz_paged.h"}"', "int main(void) {",
           '  printf("size %zu\\n", sizeof(bz_paged_kv));', '  printf("e4m3 %d\\n", BZ_KV_E4M3);']
    src += [f'  printf("{f} %zu\\n", offsetof(bz_paged_kv, {f}));' for f in fields] + ["  return 0;", "}"]
    c, exe = tmp_path / "layout.c", tmp_path / "layout"
    c.write_text("\n".join(src))
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", str(c), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(_lib.PagedKv) and int(got["e4m3"]) == _lib.KV_E4M3
    for f in fields:
        assert int(got[f]) == getattr(_lib.PagedKv, f).offset, f


FAKE = 1 << 20  # never dereferenced: every case fails validation


def _desc(**kw):
    d = _lib.PagedKv()
    ok = {"abi_version": _lib.ABI_VERSION, "T": 3, "B": 3, "HQ": 4, "HKV": 2, "D": 64, "kv_dtype": _lib.DT_BF16,
          "page_size": 16, "num_pages": 8, "table_width": 2, "k_pages": FAKE, "v_pages": FAKE, "k_page": 2048,
          "k_head": 1024, "k_pos": 64, "v_page": 2048, "v_head": 1024, "v_pos": 64, "block_table": FAKE, "ld_table": 2,
          "kv_lens": FAKE}
    for k, v in (ok | kw).items():
        setattr(d, k, v)
    return d


BAD = [
    ({"abi_version": 3}, "ERR_ABI"),
    ({"T": 0}, "ERR_INVALID_ARG"),
    ({"B": 0}, "ERR_INVALID_ARG"),
    ({"HQ": 5}, "ERR_INVALID_ARG"),
    ({"HKV": 0}, "ERR_INVALID_ARG"),
    ({"num_pages": 0}, "ERR_INVALID_ARG"),
    ({"table_width": 0}, "ERR_INVALID_ARG"),
    ({"groups": -1}, "ERR_INVALID_ARG"),
    ({"groups": 1}, "ERR_INVALID_ARG"),                                    # no prefix_width
    ({"groups": 1, "prefix_width": 1, "ld_prefix": 1}, "ERR_INVALID_ARG"),  # no prefix_table
    ({"groups": 2, "prefix_width": 1, "ld_prefix": 1, "prefix_table": FAKE, "prefix_lens": FAKE}, "ERR_INVALID_ARG"),
    ({"groups": 1, "prefix_width": 2, "ld_prefix": 1, "prefix_table": FAKE, "prefix_lens": FAKE}, "ERR_SHAPE"),
    ({"kv_dtype": _lib.DT_F32}, "ERR_INVALID_ARG"),
    ({"kv_dtype": _lib.KV_E4M3}, "ERR_INVALID_ARG"),                       # no scales
    ({"k_scale": FAKE}, "ERR_INVALID_ARG"),                                # scales of a bf16 cache
    ({"D": 96}, "ERR_UNSUPPORTED"),
    ({"D": 512}, "ERR_UNSUPPORTED"),
    ({"HQ": 34}, "ERR_UNSUPPORTED"),                                       # 17 heads of one
    ({"page_size": 8}, "ERR_UNSUPPORTED"),
    ({"page_size": 48}, "ERR_UNSUPPORTED"),
    ({"page_size": 8192}, "ERR_UNSUPPORTED"),
    ({"table_width": 1 << 27, "ld_table": 1 << 27}, "ERR_UNSUPPORTED"),
    ({"groups": 1, "prefix_width": 1 << 27}, "ERR_UNSUPPORTED"),
    ({"T": 1 << 29, "q_starts": FAKE}, "ERR_UNSUPPORTED"),
    ({"k_pages": None}, "ERR_INVALID_ARG"),
    ({"block_table": None}, "ERR_INVALID_ARG"),
    ({"kv_lens": None}, "ERR_INVALID_ARG"),
    ({"T": 4}, "ERR_SHAPE"),                                               # rows without q_starts
    ({"ld_table": 1}, "ERR_SHAPE"),
    ({"k_pos": 32}, "ERR_SHAPE"),
    ({"v_head": 0}, "ERR_SHAPE"),
    ({"v_page": 2052}, "ERR_ALIGNMENT"),
    ({"k_pages": FAKE + 8}, "ERR_ALIGNMENT"),
    ({"k_pos": 1 << 30}, "ERR_UNSUPPORTED"),
]


@pytest.mark.parametrize("kw,status", BAD)
def test_c_refuses_a_cache(kw, status):
    d, L = _desc(**kw), _lib.lib()
    want = getattr(_lib, status)
    assert L.bz_paged_attn(d, FAKE, 256, 0.1, None, 0, FAKE, 256, None) == want
    assert L.bz_paged_rope_cache(d, FAKE, 512, None, None, 1e-6, FAKE, FAKE, _lib.DT_F32, 64, 5, None, FAKE, 256,
                                 None) == want


@pytest.mark.parametrize("args,status", [
    ((None, 256, 0.1, None, 0, FAKE, 256), "ERR_INVALID_ARG"),
    ((FAKE, 256, 0.1, None, 0, None, 256), "ERR_INVALID_ARG"),
    ((FAKE, 256, 0.0, None, 0, FAKE, 256), "ERR_INVALID_ARG"),
    ((FAKE, 256, -1.0, None, 0, FAKE, 256), "ERR_INVALID_ARG"),
    ((FAKE, 256, float("nan"), None, 0, FAKE, 256), "ERR_INVALID_ARG"),
    ((FAKE, 256, float("inf"), None, 0, FAKE, 256), "ERR_INVALID_ARG"),
    ((FAKE, 248, 0.1, None, 0, FAKE, 256), "ERR_SHAPE"),
    ((FAKE, 256, 0.1, None, 0, FAKE, 192), "ERR_SHAPE"),
    ((FAKE + 2, 256, 0.1, None, 0, FAKE, 256), "ERR_ALIGNMENT"),
    ((FAKE, 260, 0.1, None, 0, FAKE, 256), "ERR_ALIGNMENT"),
    ((FAKE, 256, 0.1, None, 0, FAKE + 8, 256), "ERR_ALIGNMENT"),
    ((FAKE, 256, 0.1, None, 0, FAKE, 257), "ERR_ALIGNMENT"),
])
def test_c_refuses_attention(args, status):
    assert _lib.lib().bz_paged_attn(_desc(), *args, None) == getattr(_lib, status)


@pytest.mark.parametrize("kw,status", [
    ({"qkv": None}, "ERR_INVALID_ARG"),
    ({"cos": None}, "ERR_INVALID_ARG"),
    ({"q": None}, "ERR_INVALID_ARG"),
    ({"qn": FAKE}, "ERR_INVALID_ARG"),
    ({"dt": 2}, "ERR_INVALID_ARG"),
    ({"ld": 504}, "ERR_SHAPE"),
    ({"ldq": 128}, "ERR_SHAPE"),
    ({"ldc": 32}, "ERR_SHAPE"),
    ({"rows": 0}, "ERR_SHAPE"),
    ({"qkv": FAKE + 4}, "ERR_ALIGNMENT"),
    ({"sin": FAKE + 4}, "ERR_ALIGNMENT"),
    ({"ld": 513}, "ERR_ALIGNMENT"),
    ({"ldc": 65}, "ERR_ALIGNMENT"),
    ({"pos": FAKE + 4}, "ERR_ALIGNMENT"),
])
def test_c_refuses_append(kw, status):
    a = {"qkv": FAKE, "ld": 512, "qn": None, "kn": None, "cos": FAKE, "sin": FAKE, "dt": _lib.DT_F32, "ldc": 64,
         "rows": 5, "pos": None, "q": FAKE, "ldq": 256} | kw
    rc = _lib.lib().bz_paged_rope_cache(_desc(), a["qkv"], a["ld"], a["qn"], a["kn"], 1e-6, a["cos"], a["sin"], a["dt"],
                                        a["ldc"], a["rows"], a["pos"], a["q"], a["ldq"], None)
    assert rc == getattr(_lib, status)


def test_workspace_of_refused_sizes():
    assert _lib.lib().bz_paged_attn_workspace(_desc(D=96)) == 0
    assert _lib.lib().bz_paged_attn_workspace(None) == 0


def _served_on(monkeypatch, call):
    """The wrapper's way to the library on CPU tensors: `call` stands for the launches, the thread's name for its
    stream; a workspace for each stream, as ever."""
    monkeypatch.setattr(paged, "_gpu", lambda *a: None)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: int(threading.current_thread().name))
    monkeypatch.setattr(_lib, "capture_of", lambda stream: None)
    monkeypatch.setattr(paged, "_call", lambda index, stream, f, *args: call(stream, args))
    monkeypatch.setattr(paged, "_WS", {})


def _in_threads(streams, f):
    errors = []

    def work():
        try:
            f()
        except BaseException as e:  # noqa: BLE001 - handed to the test
            errors.append(e)

    threads = [threading.Thread(target=work, name=str(s)) for s in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


def test_threads_of_one_stream_call_one_after_the_other(monkeypatch):
    """A call can be two launches, the second of which reads what the first left in the stream's workspace: no
    other call may come between them."""
    inside, most = [], []

    def call(stream, args):
        inside.append(args[4])  # the workspace
        most.append(max(inside.count(w) for w in inside))
        time.sleep(0.005)
        inside.remove(args[4])

    _served_on(monkeypatch, call)
    a = _args(prefix_table=torch.zeros(1, dtype=torch.int32), prefix_lens=torch.zeros(1, dtype=torch.int32))
    _in_threads([1, 1, 1, 1], lambda: [paged.shared_prefix_attention(**a) for _ in range(5)])
    assert len(most) == 20 and max(most) == 1


def test_threads_of_two_streams_do_not_wait_for_each_other(monkeypatch):
    together = threading.Barrier(2, timeout=20)
    _served_on(monkeypatch, lambda stream, args: together.wait())
    a = _args()
    _in_threads([1, 2], lambda: paged.paged_attention(**a))


# A grid's dimension has less than 2^32 threads, 256 or 512 to a workgroup.
TOO_MANY = [
    # a workgroup for each row of the joining launch
    {"T": 1 << 24, "q_starts": FAKE},
    {"T": (1 << 24) + 5, "HQ": 2, "HKV": 1, "q_starts": FAKE, "groups": 1, "prefix_width": 1, "ld_prefix": 1,
     "prefix_table": FAKE, "prefix_lens": FAKE, "table_width": 1},
    # a workgroup for each tile and key/value head
    {"T": 1 << 23, "B": 1 << 23, "table_width": 1, "ld_table": 1, "HQ": 4, "HKV": 4},
]


@pytest.mark.parametrize("kw", TOO_MANY)
def test_c_refuses_more_workgroups_than_a_grid_has(kw):
    d, L = _desc(**({"table_width": 64, "ld_table": 64} | kw)), _lib.lib()
    width = d.HQ * d.D
    assert L.bz_paged_attn(d, FAKE, width, 0.1, None, 0, FAKE, width, None) == _lib.ERR_UNSUPPORTED
    assert L.bz_paged_attn_workspace(d) == 0


def test_workspace_of_as_many_rows_as_there_can_be():
    L = _lib.lib()
    assert L.bz_paged_attn_workspace(_desc(T=(1 << 24) - 1, q_starts=FAKE, table_width=64, ld_table=64)) > 0
    # positions for one chunk: no parts to be joined
    assert L.bz_paged_attn_workspace(_desc(T=1 << 24, B=1 << 20, HQ=1, HKV=1, q_starts=FAKE, table_width=8)) > 0


@pytest.mark.parametrize("T", [1 << 24, (1 << 24) + 1])
def test_c_refuses_append_of_more_rows_than_a_grid_has(T):
    d = _desc(T=T, q_starts=FAKE)
    assert _lib.lib().bz_paged_rope_cache(d, FAKE, 512, None, None, 1e-6, FAKE, FAKE, _lib.DT_F32, 64, 5, None, FAKE, 256,
                                          None) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("one_part", [0.5, 0.50390625])
def test_bound_of_two_parts_tells_them_from_one(one_part):
    """One bf16 part of the probabilities of tests/_paged_parts.midway, rounded down (or cut) or up."""
    ref = np.full((1, 1, 64), VALUE)
    total = 1 + (KEYS - 1) * PROB
    bound = parts_bound(ref, ref, np.full((1, 1), -np.log(PROB)), 64, KEYS)
    wrong = torch.tensor(VALUE * (1 + (KEYS - 1) * one_part) / total).to(BF16).double().item()
    assert (abs(wrong - ref) > bound).all()
    first, rest = 0.5, PROB - 0.5  # (both bf16 numbers)
    assert (abs(VALUE * (1 + (KEYS - 1) * (first + rest)) / total - ref) <= bound).all()
    assert half_step(1.75) == half_step(1.0) == 2.0 ** -8 and half_step(2.0) == 2.0 ** -7 and half_step(0.9) == 2.0 ** -9
