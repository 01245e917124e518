"""What the fronts of the attention side refuse of CUDA tensors (nothing is launched)."""
from __future__ import annotations

import copy

import pytest
import torch

from conftest import load_pkg

pkg = load_pkg()
pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def cache():
    return pkg.kvcache.KVCache4(4, 2, 64, page_size=16)


def rows(T, H, D=64, dtype=torch.bfloat16, device="cuda"):
    return torch.zeros(T, H, D, dtype=dtype, device=device)


def test_rotary():
    rot = pkg.rotary.AxisRotary(64, sections=(16, 16))
    q, k, pos = rows(3, 4), rows(3, 2), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    g = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for args, kw in (((q[0], k, pos), {}), ((q, k[:2], pos), {}), ((q, k.half(), pos), {}), ((q, rows(3, 2, 128), pos), {}),
                     ((q, k, pos.float()), {}), ((q, k, pos.cpu()), {}), ((q, k, pos[:, :2]), {}), ((q, k, pos.T), {}),
                     ((q, k, pos), dict(q_gain=g)), ((q, k, pos), dict(q_gain=g, k_gain=g.float())),
                     ((q, k, pos), dict(q_gain=g[:32], k_gain=g))):
        with pytest.raises(ValueError):
            rot(*args, **kw)
    with pytest.raises(TypeError):
        rot(q.float(), k.float(), pos)
    with pytest.raises(RuntimeError, match="autograd"):
        rot(q.clone().requires_grad_(), k, pos)
    with pytest.raises(pkg._lib.LibraryError, match="rotary_dim"):
        pkg.rotary.AxisRotary(128)(q, k, pos[0])
    with pytest.raises(pkg._lib.LibraryError, match="head_dim"):
        rot(rows(3, 2, 96), rows(3, 2, 96), pos)


def test_cache_rows(cache):
    k, v, s = rows(3, 2), rows(3, 2), torch.zeros(3, **INT)
    for args in ((k[:2], v, s), (k, v[:2], s), (k, v, s[:2]), (k, v, s.long()), (k, v, s.cpu()), (rows(3, 1), v, s),
                 (rows(3, 2, 128), v, s), (k.half(), v, s), (k, v, s[None])):
        with pytest.raises(ValueError):
            cache.write(*args)
    with pytest.raises(TypeError):
        cache.write(k.float(), v, s)
    with pytest.raises(RuntimeError):
        cache.write(k.cpu(), v, s)
    with pytest.raises(RuntimeError, match="autograd"):
        cache.write(k, v.clone().requires_grad_(), s)
    for bad in (s.long(), s.cpu(), s[None]):
        with pytest.raises(ValueError):
            cache.read(bad)
    with pytest.raises(TypeError):
        copy.deepcopy(cache)


def test_step_plan():
    i, t = torch.zeros(3, **INT), torch.zeros(3, 2, **INT)
    plan = pkg.kvcache.plan_step
    for args in ((i, i[:2], t, i, i[:1]), (i, i, t[:2], i, i[:1]), (i, i, t, i, i), (i, i, t, i.long(), i[:1]),
                 (i, i, t, i.cpu(), i[:1]), (i[None], i, t, i, i[:1]), (i, i, t.long(), i, i[:1]), (i, i, t.T.contiguous().T, i, i[:1]),
                 (i[:0], i[:0], t[:0], i, i[:1]), (i, i, t[:, :0], i, i[:1])):
        with pytest.raises(ValueError):
            plan(*args, page_size=16, max_tokens=4)
    for kw in (dict(page_size=24, max_tokens=4), dict(page_size=16, max_tokens=0)):
        with pytest.raises(ValueError):
            plan(i, i, t, i, i[:1], **kw)


def test_attend(cache):
    q, t, n, s = rows(3, 4), torch.zeros(3, 2, **INT), torch.ones(3, **INT), torch.arange(4, **INT)
    for args, kw in (((rows(3, 3), t, n), {}), ((q[0], t, n), {}), ((rows(3, 4, 128), t, n), {}), ((q.half(), t, n), {}),
                     ((q, t.long(), n), {}), ((q, t.cpu(), n), {}), ((q, t[0], n), {}), ((q, t, n[:2]), {}), ((q, t, n.long()), {}),
                     ((q, t[:2], n[:2]), {}), ((q, t, n, s[:3]), {}), ((q, t, n, s.long()), {}), ((q, t[:, :0], n), {}),
                     ((q, t, n), dict(window=-1)), ((q, t, n), dict(sinks=-1)), ((q, t, n), dict(scale=float("nan"))),
                     ((q, t, n), dict(gate=q[:2])), ((q, t, n), dict(gate=q.half())), ((q, t, n), dict(out=q[:2])),
                     ((q, t, n), dict(out=q.half())), ((q, t, n), dict(out=rows(3, 4, 65)[..., 1:])),
                     ((rows(3, 130), t, n), {})):
        with pytest.raises(ValueError):
            cache.attend(*args, **kw)
    with pytest.raises(TypeError):
        cache.attend(q.float(), t, n)
    with pytest.raises(RuntimeError, match="autograd"):
        cache.attend(q.clone().requires_grad_(), t, n)
    with torch.no_grad():
        assert not cache.attend(q.clone().requires_grad_(), t, n).any()
    assert cache.attend(q[:0], t[:0], n[:0]).shape == (0, 4, 64)
