"""What the attention side refuses, on the CPU: the Python fronts' checks, and the C entries' (which answer
before they touch a device)."""
from __future__ import annotations

import copy
import ctypes
import pickle
import types

import pytest
import torch

from conftest import load_pkg

pkg = load_pkg()
L = pkg._lib.lib()
ROOM = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(ROOM) + 15) & ~15


def message():
    return L.b200lut_last_error().decode()


def refused(rc, code, text):
    assert rc == code and text in message(), (rc, message())


def test_axis_rotary_arguments():
    R = pkg.rotary.AxisRotary
    for bad in (dict(rotary_dim=8), dict(rotary_dim=40), dict(rotary_dim=512), dict(rotary_dim=64, theta=0.0),
                dict(rotary_dim=64, theta=float("inf")), dict(rotary_dim=64, sections=(16, 8)), dict(rotary_dim=64, sections=()),
                dict(rotary_dim=64, sections=(40, -8)), dict(rotary_dim=64, sections=(4, 24, 4), interleaved=True)):
        with pytest.raises(ValueError):
            R(**bad)
    rot = R(64, theta=1e6, sections=(12, 10, 10), interleaved=True)
    assert rot.axes == 3 and [rot.axis.tolist().count(a) for a in range(3)] == [12, 10, 10]
    assert rot.axis[:6].tolist() == [0, 1, 2, 0, 1, 2]
    assert R(32, sections=(10, 6)).axis.tolist() == [0] * 10 + [1] * 6
    for other in (copy.deepcopy(rot), pickle.loads(pickle.dumps(rot))):
        assert torch.equal(other.axis, rot.axis) and torch.equal(other.turns, rot.turns)
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        rot(x, x, torch.arange(2))


def test_cache_arguments():
    C = pkg.kvcache.KVCache4
    for bad in (dict(page_size=48), dict(page_size=8), dict(page_size=512), dict(head_dim=96), dict(n_pages=0),
                dict(n_kv_heads=0), dict(n_kv_heads=5000), dict(n_pages=2 ** 27, page_size=16)):
        with pytest.raises(ValueError):
            C(**{**dict(n_pages=4, n_kv_heads=2, head_dim=64), **bad})
    with pytest.raises(TypeError):
        C(4, 2, 64, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="CUDA"):
        C(4, 2, 64, device="cpu")


def test_step_plan_arguments():
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.kvcache.plan_step(i, i, torch.zeros(3, 2, dtype=torch.int32), i, i[:1], page_size=16, max_tokens=4)


def cache_view(**kw):
    d = dict(k_codes=AT, v_codes=AT, k_pairs=AT, v_pairs=AT, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, dtype=0)
    d.update(kw)
    return pkg._lib.KVCacheView(**d)


@pytest.mark.parametrize("kw,code,text", [
    (dict(k_codes=None), 1, "null cache"), (dict(v_pairs=None), 1, "null cache"), (dict(dtype=2), 1, "dtype"),
    (dict(head_dim=96), 2, "head_dim"), (dict(page_size=24), 2, "page_size"), (dict(page_size=512), 2, "page_size"),
    (dict(page_size=8), 2, "page_size"), (dict(n_kv_heads=0), 1, "heads"), (dict(n_pages=0), 1, "slots"),
    (dict(n_pages=2 ** 27), 1, "2^31"), (dict(v_codes=AT + 8), 5, "16-byte"), (dict(k_pairs=AT + 4), 5, "16-byte")])
def test_c_cache_views(kw, code, text):
    v = cache_view(**kw)
    refused(L.b200lut_kv_write(ctypes.byref(v), AT, AT, 128, 64, 128, 64, AT, 1, None), code, text)
    refused(L.b200lut_kv_read(ctypes.byref(v), AT, AT, AT, 1, None), code, text)
    a = pkg._lib.AttendArgs(cache=ctypes.pointer(v))
    refused(L.b200lut_attend(ctypes.byref(a), AT, 1 << 30, None), code, text)


def test_c_write_and_read():
    v = cache_view()
    w, r = L.b200lut_kv_write, L.b200lut_kv_read
    refused(w(None, AT, AT, 128, 64, 128, 64, AT, 1, None), 1, "null cache")
    refused(w(ctypes.byref(v), None, AT, 128, 64, 128, 64, AT, 1, None), 1, "null argument")
    refused(w(ctypes.byref(v), AT, AT, 128, 64, 128, 64, None, 1, None), 1, "null argument")
    refused(w(ctypes.byref(v), AT, AT, 128, 64, 128, 64, AT, -1, None), 1, "null argument")
    for strides in ((127, 64, 128, 64), (128, 60, 128, 64), (128, 64, 4, 64), (128, 64, 128, 1)):
        refused(w(ctypes.byref(v), AT, AT, *strides, AT, 1, None), 5, "16-byte")
    refused(w(ctypes.byref(v), AT + 2, AT, 128, 64, 128, 64, AT, 1, None), 5, "16-byte")
    refused(r(ctypes.byref(v), AT, AT + 8, AT, 1, None), 5, "16-byte")
    refused(r(ctypes.byref(v), AT, None, AT, 1, None), 1, "null argument")
    assert w(ctypes.byref(v), None, None, 128, 64, 128, 64, None, 0, None) == 0
    assert r(ctypes.byref(v), None, None, None, 0, None) == 0


def test_c_plan():
    def args(**kw):
        d = {n: AT for n, _ in pkg._lib.KVPlanArgs._fields_[:11]}
        d.update(B=2, width=2, free_count=2, page_size=16, max_tokens=8)
        d.update(kw)
        return ctypes.byref(pkg._lib.KVPlanArgs(**d))
    refused(L.b200lut_kv_plan(None, None), 1, "null")
    for name, _ in pkg._lib.KVPlanArgs._fields_[:11]:
        refused(L.b200lut_kv_plan(args(**{name: None}), None), 1, "null")
    refused(L.b200lut_kv_plan(args(B=0), None), 2, "requests")
    refused(L.b200lut_kv_plan(args(B=8193), None), 2, "requests")
    refused(L.b200lut_kv_plan(args(width=0), None), 1, "width")
    refused(L.b200lut_kv_plan(args(free_count=-1), None), 1, "free_count")
    refused(L.b200lut_kv_plan(args(max_tokens=0), None), 1, "max_tokens")
    refused(L.b200lut_kv_plan(args(page_size=20), None), 2, "page_size")


def test_c_rotary():
    def args(**kw):
        d = {n: AT for n in ("q", "k", "q_out", "k_out", "positions", "turns", "axis")}
        d.update(q_token_stride=128, q_head_stride=64, k_token_stride=64, k_head_stride=64, pos_stride=0, T=1, n_heads=2,
                 n_kv_heads=1, D=64, R=64, pos64=0, dtype=0, eps=1e-6)
        d.update(kw)
        return ctypes.byref(pkg._lib.RotaryArgs(**d))
    refused(L.b200lut_rotary(None, None), 1, "null")
    for name in ("q", "k", "q_out", "k_out", "positions", "turns", "axis"):
        refused(L.b200lut_rotary(args(**{name: None}), None), 1, "null")
    refused(L.b200lut_rotary(args(dtype=2), None), 1, "dtype")
    refused(L.b200lut_rotary(args(D=96), None), 2, "head_dim")
    for R in (0, 8, 24, 80):
        refused(L.b200lut_rotary(args(R=R), None), 2, "rotary_dim")
    refused(L.b200lut_rotary(args(T=-1), None), 1, "T >= 0")
    refused(L.b200lut_rotary(args(n_heads=0), None), 1, "heads")
    refused(L.b200lut_rotary(args(q_gain=AT), None), 1, "together")
    refused(L.b200lut_rotary(args(pos_stride=-1), None), 1, "pos_stride")
    for name in ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride"):
        refused(L.b200lut_rotary(args(**{name: 4}), None), 5, "16-byte")
    refused(L.b200lut_rotary(args(k_out=AT + 2), None), 5, "16-byte")
    refused(L.b200lut_rotary(args(q_gain=AT + 2, k_gain=AT), None), 5, "16-byte")
    assert L.b200lut_rotary(args(T=0), None) == 0


def test_c_attend():
    v = cache_view()

    def args(**kw):
        d = {n: AT for n in ("q", "out", "block_table", "kv_len", "row_start")}
        d.update(cache=ctypes.pointer(v), q_token_stride=256, q_head_stride=64, out_token_stride=256, out_head_stride=64,
                 table_stride=2, T=3, B=2, width=2, n_heads=4, window=0, sinks=0, scale=0.125)
        d.update(kw)
        return ctypes.byref(pkg._lib.AttendArgs(**d))
    call = L.b200lut_attend
    big = 1 << 30
    refused(call(None, AT, big, None), 1, "null")
    for name in ("q", "out", "block_table", "kv_len"):
        refused(call(args(**{name: None}), AT, big, None), 1, "null argument")
    refused(call(args(n_heads=3), AT, big, None), 1, "multiple")
    refused(call(args(n_heads=0), AT, big, None), 1, "multiple")
    refused(call(args(n_heads=130), AT, big, None), 2, "64 query heads")
    for kw in (dict(window=-1), dict(sinks=-1), dict(width=0), dict(B=65537)):
        refused(call(args(**kw), AT, big, None), 1, "window")
    refused(call(args(T=-1), AT, big, None), 1, "negative")
    refused(call(args(row_start=None), AT, big, None), 1, "one row per request")
    for kw in (dict(q=AT + 2), dict(out=AT + 8), dict(gate=AT + 4), dict(q_token_stride=12), dict(q_head_stride=4),
               dict(out_token_stride=260), dict(out_head_stride=2), dict(gate=AT, gate_token_stride=3)):
        refused(call(args(**kw), AT, big, None), 5, "16-byte")
    refused(call(args(), None, big, None), 4, "workspace")
    refused(call(args(), AT, 64, None), 4, "workspace")
    refused(call(args(T=1 << 30), AT, big, None), 2, "too many rows")
    assert call(args(T=0), None, 0, None) == 0 and call(args(B=0), None, 0, None) == 0
    assert L.b200lut_attend_workspace_bytes(16, 4, 256, 0) > L.b200lut_attend_workspace_bytes(16, 4, 256, 1) > 0
    for bad in ((0, 1, 64), (4, 3, 64), (4, 0, 64), (4, 2, 96)):
        assert L.b200lut_attend_workspace_bytes(*bad, 1) == 0


def test_module_arguments():
    def lin(n, k=256):
        return types.SimpleNamespace(N=n, K=k)

    def qkv(q, k, v):
        return types.SimpleNamespace(q_proj=lin(q), k_proj=lin(k), v_proj=lin(v))
    rot = pkg.rotary.AxisRotary(64)
    good = dict(qkv=qkv(512, 128, 128), o_proj=lin(256, 256), rotary=rot, head_dim=64, gated=True)
    attn = pkg.PalettizedAttention(**good)
    assert (attn.n_heads, attn.n_kv_heads, attn.head_dim) == (4, 2, 64)
    g = torch.ones(64)
    for kw, text in ((dict(head_dim=96), "head_dim must be"), (dict(qkv=qkv(512, 128, 64)), "do not make"),
                     (dict(qkv=qkv(384, 128, 128)), "do not make"), (dict(qkv=qkv(512, 96, 96)), "do not make"),
                     (dict(qkv=qkv(65 * 128, 64, 64)), "do not make"), (dict(gated=False), "o_proj reads"),
                     (dict(rotary=pkg.rotary.AxisRotary(128)), "larger than head_dim"), (dict(q_gain=g), "come together"),
                     (dict(q_gain=g, k_gain=torch.ones(32)), "k_gain must be"), (dict(window=-1), "not be negative")):
        with pytest.raises(ValueError, match=text):
            pkg.PalettizedAttention(**{**good, **kw})
