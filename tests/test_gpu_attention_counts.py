"""Whether attention over the 4-bit cache counts every token once, on the GPU: equal scores, and values by which a result
moves out of its bound when 16 tokens are missing (test_attention_bounds.py), over rows that many blocks share."""
from __future__ import annotations

import pytest
import torch

from conftest import load_pkg
from helpers_attention import close, values64
from helpers_attention_tight import attend_tight, counted_values, counted_want
from test_gpu_attend import Batch

pkg = load_pkg()
pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")


def counted_batch(lengths, rows, G, H, D, page, dtype):
    """A batch in which head h has counted_values turned by 3 h elements, pages in no order."""
    g = torch.Generator(device="cuda").manual_seed(sum(lengths))
    counts = [-(-n // page) for n in lengths]
    cache = pkg.kvcache.KVCache4(sum(counts) + 1, H, D, page_size=page, dtype=dtype)
    order = torch.randperm(cache.n_pages, device="cuda", generator=g).int()
    table, at = torch.full((len(lengths), max(counts) + 1), -1, **INT), 0
    v = counted_values(max(lengths), D).cuda()
    v = torch.stack([v.roll(3 * h, 1) for h in range(H)], 1)
    for b, n in enumerate(lengths):
        table[b, :counts[b]] = order[at:at + counts[b]]
        at += counts[b]
        slots = (table[b, :counts[b]].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:n].int()
        k = torch.randn(n, H, D, device="cuda", generator=g).to(dtype)
        cache.write(k, v[:n].to(dtype), slots)
    start = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **INT)
    q = torch.zeros(sum(rows), G * H, D, dtype=dtype, device="cuda")
    return cache, q, table, torch.tensor(lengths, **INT), start, v


def check(lengths, rows, G, H, D, page, dtype):
    cache, q, table, n, start, v = counted_batch(lengths, rows, G, H, D, page, dtype)
    y = cache.attend(q, table, n, None if max(rows) == 1 else start)
    t = 0
    for length, r in zip(lengths, rows):
        ends = torch.arange(length - r + 1, length + 1, device="cuda")
        for h in range(H):
            want, tol = counted_want(v[:, h], ends, dtype)
            got = y[t:t + r, h * G:(h + 1) * G]
            close(got, want[:, None].expand_as(got), tol[:, None].expand_as(got), f"{length} tokens, head {h}")
        t += r
    assert pkg._lib.lib().b200lut_device_status() == 0


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("G,H,D,page", [(4, 4, 256, 64), (8, 1, 128, 16), (1, 2, 64, 64), (12, 1, 256, 32), (64, 1, 128, 16)])
def test_single_rows(G, H, D, page, dtype):
    check([70_001], [1], G, H, D, page, dtype)
    check([16, 40_000, 777, 1, 9001, 33], [1] * 6, G, H, D, page, dtype)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("G,H,D,page", [(4, 2, 256, 64), (8, 1, 128, 16), (1, 2, 64, 64), (12, 1, 64, 32)])
def test_chunks_and_prompts(G, H, D, page, dtype):
    check([70_001], [130], G, H, D, page, dtype)
    check([40_000, 3, 17_000, 500, 128], [2, 1, 64, 500, 9], G, H, D, page, dtype)
    check([3000], [3000], G, H, D, page, dtype)


@pytest.mark.parametrize("rows", (1, 70))
@pytest.mark.parametrize("window,sinks", [(16, 0), (1000, 16), (20_000, 4096)])
def test_windows_with_sinks(window, sinks, rows):
    n, dtype = 50_000, torch.bfloat16
    cache, q, table, length, start, v = counted_batch([n], [rows], 4, 2, 128, 16, dtype)
    y = cache.attend(q, table, length, start, window=window, sinks=sinks)
    below = torch.cat((torch.zeros_like(v[:1]), v.cumsum(0)))
    for r in range(rows):
        pos = n - rows + r
        want = (below[pos + 1] - below[pos + 1 - window] + below[sinks]) / (window + sinks)
        tol = (2.0 ** -11 + 2.0 ** -18) * (1 + want.abs()) + 2.0 ** -17 + 2.0 ** -8 * want.abs()
        got = y[r].view(2, 4, 128)
        close(got, want[:, None].expand_as(got), tol[:, None].expand_as(got), f"row {r}")


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("Hq,H,D", [(16, 4, 256), (8, 1, 128), (2, 2, 64)])
def test_long_rows_as_they_come(Hq, H, D, dtype):
    for lengths, rows in (([70_001], [1]), ([40_000, 3, 17_000], [2, 1, 64])):
        b = Batch(lengths, rows, Hq, H, D, 64, dtype)
        y, t = b.run(), 0
        for i, (n, r) in enumerate(zip(lengths, rows)):
            want, tol = attend_tight(b.q[t:t + r], values64(b.k[i]), values64(b.v[i]), torch.arange(n - r, n, device="cuda"), D ** -0.5)
            close(y[t:t + r], want, tol, f"request {i}")
            assert (y[t:t + r].double() - want).norm() <= 2.0 ** -8 * want.norm()
            t += r
