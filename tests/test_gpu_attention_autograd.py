"""Gradients on the attention side: it serves none, and says so wherever one would be lost."""
from __future__ import annotations

import pytest
import torch

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
