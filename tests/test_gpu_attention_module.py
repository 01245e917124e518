"""Rotary positions, step plan, 4-bit cache and attention together: the attention module between its projections,
and the full-attention layers of the stack."""
from __future__ import annotations

import importlib
import math

import pytest
import torch

from conftest import load_pkg
from helpers import Case
from helpers_attention import attend64, close, rotate64, values64

pkg = load_pkg()
kv = pkg.kvcache
st = importlib.import_module(pkg.__name__ + ".stack")
pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")


class Requests:
    """Page table and lengths of B requests, and the keys and values that each has brought so far."""

    def __init__(self, B, width, page, spare=3):
        self.page, self.cached = page, torch.zeros(B, **INT)
        self.table = torch.full((B, width), -1, **INT)
        self.free = torch.randperm(B * width + spare, device="cuda").int()
        self.taken = torch.zeros(1, **INT)
        self.k, self.v = [[] for _ in range(B)], [[] for _ in range(B)]

    def plan(self, fresh, rows):
        step = kv.plan_step(self.cached, fresh, self.table, self.free, self.taken, self.page, rows)
        self.cached.copy_(step.kv_len)
        self.taken.copy_(step.taken)
        return step


def layer(dtype, D, Hq, H, K, gated, gains, seed=0, **kw):
    per = 2 * D if gated else D
    mods = [Case(n, K, 128, 4, dtype, seed=seed + i, lut_std=0.1).module() for i, n in enumerate((Hq * per, H * D, H * D))]
    o = Case(K, Hq * D, 128, 4, dtype, seed=seed + 3).module()
    g = torch.Generator().manual_seed(seed)
    gain = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype) if gains else None for _ in range(2)]
    rot = pkg.rotary.AxisRotary(min(D, 64), theta=1e6)
    return pkg.PalettizedAttention(pkg.SplitQKV(*mods), o, rot, D, gated=gated, q_gain=gain[0], k_gain=gain[1], **kw).cuda()


def check_step(qkv, attended, attn, state, fresh, positions):
    """Each stage in 64 bits from the stage before it, as it was rounded."""
    D, Hq, H = attn.head_dim, attn.n_heads, attn.n_kv_heads
    per = 2 * D if attn.gated else D
    T = sum(fresh)
    q = qkv[:, :Hq * per].reshape(-1, Hq, per)
    k, v = (qkv[:, Hq * per + i * H * D:][:, :H * D].reshape(-1, H, D) for i in range(2))
    qr, kr = attn.rotary(q[..., :D].contiguous(), k.contiguous(), positions, attn.q_gain, attn.k_gain, attn.eps)
    for x, y, gain in ((q[..., :D], qr, attn.q_gain), (k, kr, attn.k_gain)):
        want, tol = rotate64(x[:T], positions[None, :T], attn.rotary.rotary_dim, attn.rotary.theta, attn.rotary.axis, gain, attn.eps)
        close(y[:T], want, tol, "rotation")
    t = 0
    for b, n in enumerate(fresh):
        state.k[b].append(kr[t:t + n])
        state.v[b].append(v[t:t + n].clone())          # the buffer is the next step's too
        if n:
            kk, vv = torch.cat(state.k[b]), torch.cat(state.v[b])
            pos = torch.arange(len(kk) - n, len(kk), device="cuda")
            assert torch.equal(positions[t:t + n].long(), pos)
            want, tol = attend64(qr[t:t + n], values64(kk), values64(vv), pos, D ** -0.5, attn.window, attn.sinks,
                                 q[t:t + n, :, D:] if attn.gated else None)
            close(attended[t:t + n], want, tol, f"request {b}")
        t += n
    assert not attended[t:].any()
    assert pkg._lib.lib().b200lut_device_status() == 0


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,Hq,H,gated,gains,kw", [(64, 4, 2, True, True, {}), (128, 2, 1, False, False, dict(window=20, sinks=2)),
                                                   (256, 4, 1, True, True, {})])
def test_module(D, Hq, H, gated, gains, kw, dtype):
    torch.manual_seed(D)
    K = 256
    attn = layer(dtype, D, Hq, H, K, gated, gains, **kw)
    seen = {}
    attn.qkv.register_forward_hook(lambda m, a, out: seen.__setitem__("qkv", out))
    attn.o_proj.register_forward_pre_hook(lambda m, a: seen.__setitem__("o", a[0]))
    cache = kv.KVCache4(3 * 6 + 3, H, D, page_size=16, dtype=dtype)
    state = Requests(3, 6, 16)
    for fresh, rows in (([7, 0, 40], 50), ([1, 1, 1], 3), ([1, 20, 1], 22), ([0, 0, 3], 16), ([1, 1, 1], 3), ([1, 1, 1], 3)):
        x = torch.full((rows, K), math.nan, device="cuda", dtype=dtype)
        x[:sum(fresh)] = torch.randn(sum(fresh), K, device="cuda").to(dtype)
        step = state.plan(torch.tensor(fresh, **INT), rows)
        y = attn(x, cache, state.table, step, one_row_each=fresh == [1, 1, 1])
        assert y.shape == (rows, K) and torch.equal(y, attn.o_proj(seen["o"])) and not y[sum(fresh):].any()
        check_step(seen["qkv"], seen["o"].view(rows, Hq, D), attn, state, fresh, step.positions)


def test_axes_and_positions_of_the_caller():
    attn = layer(torch.bfloat16, 128, 2, 1, 256, False, False)
    attn.rotary = pkg.rotary.AxisRotary(64, theta=1e6, sections=(12, 10, 10), interleaved=True)
    cache = kv.KVCache4(4, 1, 128, page_size=16)
    state = Requests(1, 3, 16, spare=1)
    x = torch.randn(20, 256, device="cuda").bfloat16()
    step = state.plan(torch.tensor([20], **INT), 20)
    text = attn(x, cache, state.table, step)
    assert torch.equal(attn(x, cache, state.table, step, positions=step.positions.expand(3, 20)), text)
    grid = torch.stack((torch.zeros(20, **INT), torch.arange(20, **INT) // 5, torch.arange(20, **INT) % 5))
    assert not torch.equal(attn(x, cache, state.table, step, positions=grid), text)


def test_captured_decode_of_two_layers_follows_the_eager_one():
    dtype, K, B = torch.bfloat16, 256, 3
    layers = [layer(dtype, 128, 4, 2, K, True, True, seed=10 * i) for i in range(2)]
    prompt = torch.randn(70, K, device="cuda").to(dtype)
    token = torch.randn(B, K, device="cuda").to(dtype)
    free = torch.randperm(B * 8, device="cuda").int()

    def start():
        state = Requests(B, 8, 16, spare=0)
        state.free = free
        caches = [kv.KVCache4(B * 8, 2, 128, page_size=16, dtype=dtype) for _ in layers]
        step = state.plan(torch.tensor([50, 5, 15], **INT), 70)
        for attn, cache in zip(layers, caches):
            attn(prompt, cache, state.table, step)
        return state, caches

    def decode(state, caches, ones, x):
        step = state.plan(ones, B)
        for attn, cache in zip(layers, caches):
            x = x + attn(x, cache, state.table, step, one_row_each=True)
        return x

    ones = torch.ones(B, **INT)
    eager, caches = start()
    want = [decode(eager, caches, ones, token) for _ in range(20)]
    captured, caches2 = start()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = decode(captured, caches2, ones, token)
    for w in want:
        graph.replay()
        assert torch.equal(out, w)
    assert torch.equal(eager.cached, captured.cached) and eager.cached.tolist() == [70, 25, 35]
    assert all(torch.equal(a, b) for c, d in zip(caches, caches2) for a, b in zip(c._buffers, d._buffers))
    assert pkg._lib.lib().b200lut_device_status() == 0


def test_stack_with_attention():
    stack = st.LinearStack(n_layers=4)
    state = st.AttentionState(stack, requests=3, max_len=100, page_size=16)
    full = stack.layers[3]
    shape = pkg.PalettizedAttention(full.qkv, full.o_proj, state.rotary, st.HEAD_DIM, gated=True)
    seen = Requests(3, 1, 16)

    def check(rows, fresh):
        plan = stack._plans[rows]
        attended, qkv = state.out(0, rows), plan["qkv"][full]
        positions = torch.zeros(rows, **INT)
        had = [sum(len(x) for x in s) for s in seen.k]
        at = torch.cat([torch.arange(h, h + n, **INT) for h, n in zip(had, fresh)])
        positions[:len(at)] = at
        check_step(qkv, attended, shape, seen, fresh, positions)
        got, want = plan["buffers"][13].double(), full.o_proj(attended.flatten(1)).double()
        assert (got - want).abs().max() <= 2.0 ** -7 * want.abs().max()

    for rows, fresh in ((40, [30, 0, 7]), (5, [1, 3, 1])):
        stack._plan(rows)["x"].copy_(torch.randn(rows, st.HIDDEN, device="cuda"))
        stack.step(rows, attention=state, fresh=torch.tensor(fresh, **INT))
        torch.cuda.synchronize()
        check(rows, fresh)
    x = stack._plan(3)["x"]
    x.copy_(torch.randn(3, st.HIDDEN, device="cuda"))
    stack.step(3, attention=state)
    torch.cuda.synchronize()
    check(3, [1, 1, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stack.step(3, attention=state)
    for _ in range(3):
        x.copy_(torch.randn(3, st.HIDDEN, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        check(3, [1, 1, 1])
    assert state.kv_len.tolist() == [35, 7, 12]
    # a request that is full is not served, the others are
    state.kv_len.copy_(torch.tensor([112, 7, 12], **INT))
    graph.replay()
    torch.cuda.synchronize()
    assert state.kv_len.tolist() == [112, 8, 13]
    stack.check_status()


def test_stack_with_programmatic_launches():
    stack = st.LinearStack(n_layers=8)
    x = stack._plan(4)["x"]
    rows = torch.randn(6, 4, st.HIDDEN, device="cuda").to(stack.dtype)

    def run(flags, captured):
        state, outs = st.AttentionState(stack, requests=4, max_len=40, page_size=16), []
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                stack.step(4, flags, attention=state)
        for r in rows:
            x.copy_(r)
            if captured:
                graph.replay()
            else:
                stack.step(4, flags, attention=state)
            outs.append([state.out(i, 4).clone() for i in range(2)] + [b.clone() for b in stack._plan(4)["buffers"]])
        torch.cuda.synchronize()
        return outs

    want = run(0, False)
    for captured in (False, True):
        got = run(pkg._lib.FLAG_PDL, captured)
        assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))
    stack.check_status()


def test_refusals():
    stack = st.LinearStack(n_layers=4)
    state = st.AttentionState(stack, requests=3, max_len=20)
    for call, text in ((lambda: stack.step(2, attention=state), "one row per request"),
                       (lambda: stack.step(3, fresh=torch.ones(3, **INT)), "AttentionState"),
                       (lambda: st.LinearStack(n_layers=4).step(3, attention=state), "another stack"),
                       (lambda: st.AttentionState(st.LinearStack(n_layers=1), 1, 1), "full attention"),
                       (lambda: st.AttentionState(st.LinearStack(n_layers=4, rotate=True), 1, 1), "unrotated"),
                       (lambda: st.AttentionState(stack, 0, 5), "positive")):
        with pytest.raises(ValueError, match=text):
            call()
    assert state.kv_len.tolist() == [0, 0, 0]
    attn = layer(torch.bfloat16, 64, 4, 2, 256, False, False)
    x = torch.zeros(3, 256, device="cuda", dtype=torch.bfloat16)
    cache, r = kv.KVCache4(4, 2, 64, page_size=16), Requests(3, 1, 16)
    step = r.plan(torch.ones(3, **INT), 3)
    for call, text in ((lambda: attn(x[None], cache, r.table, step), "x must be"),
                       (lambda: attn(x, kv.KVCache4(4, 1, 64, page_size=16), r.table, step), "cache holds"),
                       (lambda: attn(x, kv.KVCache4(4, 2, 64, page_size=16, dtype=torch.float16), r.table, step), "cache holds"),
                       (lambda: attn(x[:2], cache, r.table, step), "step plan"),
                       (lambda: attn(x[:2], cache, r.table, r.plan(torch.ones(3, **INT), 2), one_row_each=True), "one_row_each")):
        with pytest.raises(ValueError, match=text):
            call()
