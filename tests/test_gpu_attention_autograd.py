"""Gradients on the attention side: it serves none, and says so wherever one would be lost."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from conftest import load_pkg

pkg = load_pkg()
pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")


def rows(T, H, D=64):
    return torch.ones(T, H, D, dtype=torch.bfloat16, device="cuda")


def test_gains_that_require_grad():
    rot = pkg.rotary.AxisRotary(64)
    q, k, pos = rows(3, 4), rows(3, 2), torch.arange(3, device="cuda")
    g = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for _ in range(2):                              # the first call takes the Python route, the second the native one
        for gains in ((torch.nn.Parameter(g), g), (g, torch.nn.Parameter(g)), (torch.nn.Parameter(g),) * 2):
            with pytest.raises(RuntimeError, match="_gain requires grad"):
                rot(q, k, pos, *gains)
            with torch.no_grad():
                a = rot(q, k, pos, *gains)
            b = rot(q, k, pos, *(x.detach() for x in gains))
            assert all(torch.equal(x, y) and not x.requires_grad for x, y in zip(a, b))


def test_results_into_a_buffer_that_requires_grad():
    cache = pkg.kvcache.KVCache4(2, 2, 64, page_size=16)
    q, t, n = rows(1, 4), torch.zeros(1, 1, **INT), torch.ones(1, **INT)
    out = torch.zeros_like(q).requires_grad_()
    with pytest.raises(RuntimeError, match="out requires grad"):
        cache.attend(q, t, n, out=out)
    with torch.no_grad():
        assert cache.attend(q, t, n, out=out) is out


def test_forward_mode_tangents():
    rot = pkg.rotary.AxisRotary(64).to("cuda")
    cache = pkg.kvcache.KVCache4(2, 2, 64, page_size=16)
    q, k, g = rows(3, 4), rows(3, 2), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    pos, slots = torch.arange(3, device="cuda"), torch.arange(3, **INT)
    table, n, start = torch.zeros(1, 1, **INT), torch.full((1,), 3, **INT), torch.tensor([0, 3], **INT)
    with forward_ad.dual_level():
        def dual(x):
            return forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: rot(dual(q), k, pos), lambda: rot(q, dual(k), pos), lambda: rot(q, k, pos, dual(g), g),
                     lambda: rot(q, k, pos, g, dual(g)), lambda: cache.write(dual(k), k, slots), lambda: cache.write(k, dual(k), slots),
                     lambda: cache.attend(dual(q), table, n, start), lambda: cache.attend(q, table, n, start, gate=dual(q)),
                     lambda: cache.attend(q, table, n, start, out=dual(q.clone()))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):     # no_grad leaves forward mode on
                call()
            with torch.inference_mode():
                call()
        rot(q, k, pos)                                 # others' tangents are no matter
        cache.write(k, k, slots)
        cache.attend(q, table, n, start)
