"""Rotary positions over several axes on the GPU against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from conftest import load_pkg
from helpers_attention import close, rotate64

pkg = load_pkg()
pytestmark = pytest.mark.gpu
THETA = 1e7


def check(rot, q, k, positions, gains=None, eps=1e-6):
    kw = {} if gains is None else dict(q_gain=gains[0], k_gain=gains[1], eps=eps)
    got = rot(q, k, positions, **kw)
    pos = positions if positions.dim() == 2 else positions.expand(rot.axes, -1)
    for i, (x, y) in enumerate(zip((q, k), got)):
        assert y.shape == x.shape and y.is_contiguous() and y.dtype == x.dtype
        close(y, *rotate64(x, pos, rot.rotary_dim, rot.theta, rot.axis, None if gains is None else gains[i], eps), "qk"[i])
    return got


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("T,Hq,H,D,R,axes,inter,norm", [
    (1, 16, 4, 256, 64, 3, True, True),
    (1, 1, 1, 64, 16, 1, False, False),
    (37, 16, 4, 256, 64, 3, True, True),
    (5, 3, 1, 128, 128, 2, False, True),
    (129, 9, 3, 64, 64, 3, True, False),
    (64, 5, 5, 64, 48, 3, False, True),          # half a rotated row is 24 elements: three lanes
    (700, 32, 8, 128, 96, 3, True, False),       # many tokens: four groups of rows per warp
    (2051, 7, 1, 256, 256, 3, False, True),      # eight heads: the last warp of a token is part empty
])
def test_rotation(T, Hq, H, D, R, axes, inter, norm, dtype):
    g = torch.Generator(device="cuda").manual_seed(T + D + R)
    half = R // 2
    sections = [half - (axes - 1) * (half // axes)] + [half // axes] * (axes - 1)
    rot = pkg.rotary.AxisRotary(R, theta=THETA, sections=sections, interleaved=inter)
    q = torch.randn(T, Hq, D, device="cuda", generator=g).to(dtype)
    k = torch.randn(T, H, D, device="cuda", generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (axes, T), device="cuda", generator=g)
    gains = [(1 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dtype) for _ in range(2)] if norm else None
    check(rot, q, k, pos, gains)
    check(rot, q, k, pos.int(), gains)
    check(rot, q, k, pos[0], gains)


def test_strided_rows_and_positions():
    # queries beside their gates in one projection row, positions as a column of a wider matrix
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(33, 4 * 2 * 256 + 2 * 256, device="cuda", generator=g).bfloat16()
    q = rows[:, :2048].view(33, 4, 512)[..., :256]
    k = rows[:, 2048:].view(33, 2, 256)
    rot = pkg.rotary.AxisRotary(64, theta=THETA, sections=(12, 10, 10), interleaved=True)
    before = rows.clone()
    pos = torch.randint(0, 4096, (3, 66), device="cuda", generator=g)
    a = check(rot, q, k, pos[:, ::2])
    assert torch.equal(rows, before)
    # rows that are not 16-byte aligned are copied
    odd = torch.randn(33, 4, 257, device="cuda", generator=g).bfloat16()[..., 1:]
    check(rot, odd, k, pos[:, :33])
    # the inverse turn undoes the rotation (up to two roundings)
    back = rot(a[0], a[1], -pos[:, ::2].contiguous())
    assert ((back[0].double() - q.double()).abs() <= 2.0 ** -7 * (q.double().abs() + q.double().roll(32, -1).abs()
                                                                    + q.double().roll(-32, -1).abs())).all()


def test_extremes():
    rot = pkg.rotary.AxisRotary(64, theta=THETA)
    q, k = torch.zeros(2, 2, 64, device="cuda", dtype=torch.float16), torch.ones(2, 1, 64, device="cuda", dtype=torch.float16)
    gains = (torch.ones(64, device="cuda", dtype=torch.float16),) * 2
    pos = torch.tensor([0, 2 ** 31 - 1], device="cuda")
    a = rot(q, k, pos, *gains)
    assert not a[0].any()                         # a head of zeros: its norm divides by sqrt(eps)
    check(rot, q, k, pos)
    assert torch.equal(rot(q, k, pos)[1][0], k[0])        # position 0 turns nothing
    q[1, 1, 5] = float("nan")
    y = rot(q, k, pos)[0]
    assert y.isnan().sum() == 2 and y[1, 1, 5].isnan() and y[1, 1, 37].isnan()
    empty = rot(q[:0], k[:0], pos[:0])
    assert empty[0].shape == (0, 2, 64) and empty[1].shape == (0, 1, 64)


def test_captured_and_replayed_on_another_stream():
    rot = pkg.rotary.AxisRotary(128, theta=THETA).to("cuda")
    q = torch.randn(9, 4, 128, device="cuda").half()
    k = torch.randn(9, 1, 128, device="cuda").half()
    pos = torch.arange(9, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rot(q, k, pos)
    q.copy_(torch.randn_like(q))
    pos += 1000
    graph.replay()
    torch.cuda.synchronize()
    want = rot(q, k, pos)
    assert torch.equal(y[0], want[0]) and torch.equal(y[1], want[1])
