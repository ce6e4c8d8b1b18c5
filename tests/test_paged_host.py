"""The paged cache without a GPU: page bookkeeping, rotation tables, the argument structs and every refusal of the C
entries (which come before any CUDA call)."""
import ctypes as C
import math

import numpy as np
import pytest

import nekochat_b200 as nb
from nekochat_b200 import ops
from nekochat_b200.paged import PagedCache
from tests import paged_reference as ref

CACHE = ["k_pages", "v_pages", "k_scale", "v_scale", "table", "page_stride", "scale_stride", "table_stride", "type", "n_seq",
         "max_pages", "num_pages", "n_kv", "page_size", "head_dim", "reserved"]
APPEND = CACHE + ["q", "k", "v", "q_out", "q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "o_token", "o_head",
                  "start", "q_start", "cs", "q_gain", "k_gain", "qtype", "tokens", "n_head", "max_new", "rot", "cs_rows",
                  "interleaved", "eps"]
ATTEND = CACHE + ["q", "out", "q_token", "q_head", "o_token", "o_head", "kv_len", "q_start", "slopes", "prefix", "qtype",
                  "tokens", "n_head", "max_new", "window", "scale", "softcap", "reserved2"]
GOOD = dict(k_pages=4096, v_pages=8192, k_scale=64, v_scale=64, table=64, page_stride=8 * 16 * 128, scale_stride=8,
            table_stride=4, type=3, n_seq=2, max_pages=4, num_pages=9, n_kv=8, page_size=16, head_dim=128, reserved=0,
            q=64, k=64, v=64, q_out=64, out=64, q_token=2048, q_head=128, k_token=1024, k_head=128, v_token=1024, v_head=128,
            o_token=2048, o_head=128, start=64, q_start=64, cs=64, q_gain=64, k_gain=64, qtype=0, tokens=0, n_head=16,
            max_new=1, rot=128, cs_rows=100, interleaved=0, eps=1e-6, kv_len=64, slopes=0, prefix=0, window=0, scale=0.1,
            softcap=0.0, reserved2=0)


def call(name, fields, fmt, **over):
    """Packed arguments with tokens = 0 unless overridden: a call that passes the checks of the cache does nothing."""
    d = dict(GOOD, **over)
    return getattr(nb.lib(), name)(fmt.pack(*(d[f] for f in fields)), None)


def test_structs_match_the_header(tmp_path):
    """Python's packed layouts have the compiler's sizes and field places."""
    import os
    import subprocess
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "neko_cuda.h"\n'
                   "int main(void){printf(\"%zu %zu %zu %zu %zu %zu\\n\", sizeof(neko_paged_append_args), sizeof(neko_paged_attention_args),"
                   "offsetof(neko_paged_append_args, eps), offsetof(neko_paged_append_args, start),"
                   "offsetof(neko_paged_attention_args, kv_len), offsetof(neko_paged_attention_args, softcap));return 0;}\n")
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got[:2] == [ops._APPEND.size, ops._ATTEND.size]
    a = ops._APPEND.pack(*(GOOD[f] if f not in ("eps", "start") else (0.5 if f == "eps" else 0x1122334455) for f in APPEND))
    assert np.frombuffer(a, np.float32)[got[2] // 4] == 0.5 and np.frombuffer(a, np.int64)[got[3] // 8] == 0x1122334455
    b = ops._ATTEND.pack(*(GOOD[f] if f not in ("softcap", "kv_len") else (2.5 if f == "softcap" else 0x1122334455) for f in ATTEND))
    assert np.frombuffer(b, np.int64)[got[4] // 8] == 0x1122334455 and np.frombuffer(b, np.float32)[got[5] // 4] == 2.5


@pytest.mark.parametrize("name,fields,fmt", [("neko_op_paged_append", APPEND, ops._APPEND),
                                             ("neko_op_paged_attention", ATTEND, ops._ATTEND)])
@pytest.mark.parametrize("over", [dict(k_pages=0), dict(v_pages=0), dict(table=0), dict(k_scale=0), dict(v_scale=0), dict(type=0),
                                  dict(type=2), dict(type=7), dict(n_seq=-1), dict(max_pages=0), dict(num_pages=0), dict(n_kv=0),
                                  dict(page_size=8), dict(page_size=48), dict(page_size=256), dict(head_dim=96), dict(head_dim=256),
                                  dict(page_stride=8 * 16 * 128 - 16), dict(page_stride=8 * 16 * 128 + 8), dict(k_pages=4104),
                                  dict(v_pages=8), dict(table_stride=3), dict(scale_stride=7), dict(max_pages=1 << 27, table_stride=1 << 27),
                                  dict(qtype=3), dict(qtype=-1), dict(tokens=-1), dict(max_new=-1), dict(n_head=0)])
def test_refused_caches(name, fields, fmt, over):
    assert call(name, fields, fmt) == 0  # nothing to do, and nothing wrong
    assert call(name, fields, fmt, **over) == -1
    assert name[8:].encode() in nb.lib().neko_last_error()


@pytest.mark.parametrize("over", [dict(k=0), dict(v=0), dict(start=0), dict(q_out=0), dict(q_start=0, tokens=3), dict(rot=12),
                                  dict(rot=136), dict(rot=-8), dict(cs=0), dict(cs_rows=0), dict(cs=72), dict(q_gain=0),
                                  dict(k_gain=0)])
def test_refused_appends(over):
    assert call("neko_op_paged_append", APPEND, ops._APPEND, **dict(dict(tokens=2), **over)) == -1


@pytest.mark.parametrize("over", [dict(q=0), dict(out=0), dict(kv_len=0), dict(q_start=0, tokens=3), dict(n_head=12), dict(window=-1),
                                  dict(softcap=-1.0), dict(softcap=math.nan), dict(scale=math.nan)])
def test_refused_attentions(over):
    assert call("neko_op_paged_attention", ATTEND, ops._ATTEND, **dict(dict(tokens=2), **over)) == -1
    assert call("neko_op_paged_attention", ATTEND, ops._ATTEND, tokens=2, n_seq=20000) == -6


@pytest.mark.parametrize("over", [dict(k_token=1 << 24), dict(v_token=-(1 << 24)), dict(q_token=1 << 40), dict(o_token=1 << 24)])
def test_refused_token_strides(over):
    assert call("neko_op_paged_append", APPEND, ops._APPEND, **dict(dict(tokens=2), **over)) == -6
    assert b"token strides" in nb.lib().neko_last_error()


def test_null_arguments():
    assert nb.lib().neko_op_paged_append(None, None) == -1
    assert nb.lib().neko_op_paged_attention(None, None) == -1


def test_pages_are_handed_out_and_given_back():
    import torch
    c = PagedCache(1, 2, 32, pages=6, page=16, kind="f16", max_seqs=3, max_len=64, device="cpu")
    assert c.pool.dtype == torch.float16 and c.layer(0)[2] is None
    a, b = c.open(), c.open()
    c.grow([(a, 17), (b, 16)])
    c.length[a], c.length[b] = 17, 16
    assert [len(c.held[a]), len(c.held[b]), len(c.free)] == [2, 1, 3]
    c.grow([(a, 15), (b, 1)])
    assert [len(c.held[a]), len(c.held[b])] == [2, 2]
    t = c.rows([b, a])
    assert t.shape == (2, 2) and len(set(t.ravel())) == 4 and (t >= 0).all()
    with pytest.raises(nb.NekoError):
        c.grow([(a, 48)])              # past max_len
    c.length[a] = 32
    with pytest.raises(nb.NekoError):
        c.grow([(a, 32), (b, 33)])     # more pages than there are: nothing changes
    assert [len(c.held[a]), len(c.held[b]), len(c.free)] == [2, 2, 2]
    d = c.open()
    with pytest.raises(nb.NekoError):
        c.open()
    c.close(a), c.close(d), c.close(b)
    assert sorted(c.free) == list(range(6)) and not c.held and len(c.ids) == 3
    with pytest.raises(nb.NekoError):
        PagedCache(1, 2, 32, pages=6, kind="int4", device="cpu")


def test_rotation_tables():
    plain = ops.rope_table(100, 64, 1e4, device="cpu").numpy()
    ang = np.arange(100)[:, None] * 1e4 ** (-np.arange(32) / 32)
    assert np.array_equal(plain, np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32))
    linear = ops.rope_table(400, 64, 1e4, "linear", 4.0, device="cpu").numpy()
    assert np.allclose(linear[::4], plain, atol=1e-6)
    ntk = ops.rope_table(100, 64, 1e4, "ntk", 4.0, device="cpu").numpy()
    assert np.array_equal(ntk[:, 0], plain[:, 0])                               # the fastest pair keeps its speed
    slow = lambda t: np.arctan2(t[1:, -1, 1], t[1:, -1, 0])  # noqa: E731
    assert np.allclose(slow(ntk), slow(plain) / 4, rtol=1e-4)                    # the slowest is slowed by the factor
    yarn = ops.rope_table(100, 64, 1e4, "yarn", 4.0, 32, beta_fast=4.0, device="cpu").numpy()
    gain = 0.1 * math.log(4.0) + 1
    assert np.allclose(np.hypot(yarn[..., 0], yarn[..., 1]), gain, rtol=1e-6)
    assert np.allclose(yarn[:, 0], gain * plain[:, 0], atol=1e-6) and np.allclose(slow(yarn), slow(plain) / 4, rtol=1e-4)
    for bad in (dict(rot=12), dict(rot=0), dict(positions=0), dict(scaling="yarn"), dict(scaling="other"), dict(factor=0.5)):
        with pytest.raises(nb.NekoError):
            ops.rope_table(**{**dict(positions=4, rot=64, theta=1e4, device="cpu"), **bad})


def test_reference_codes():
    """The tests' own 8-bit rounding: exact on codes, to nearest with ties to even between them, saturating."""
    codes = ref.E4M3[np.isfinite(ref.E4M3)]
    assert len(codes) == 254 and codes.max() == 448 and np.array_equal(ref.e4m3_round(codes), codes)
    pos = np.unique(np.abs(codes))
    mid = (pos[1:] + pos[:-1]) / 2
    got = ref.e4m3_round(mid)
    lower_even = np.arange(len(mid)) % 2 == 0
    assert np.array_equal(got, np.where(lower_even, pos[:-1], pos[1:]))
    assert ref.e4m3_round(1e9) == 448 and ref.e4m3_round(-np.inf) == -448 and np.isnan(ref.e4m3_round(np.nan))
    assert ref.block_scale(np.array([448.0])) == 1 and ref.block_scale(np.array([448.1, np.inf, np.nan])) == 2
    assert ref.block_scale(np.zeros(3)) == 2.0 ** -100
