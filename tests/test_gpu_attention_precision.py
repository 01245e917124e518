"""What a row's result may depend on, and how closely: attention on the GPU against bounds from the row's own weights."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import load_pkg
from helpers_attention import close, values64
from helpers_attention_tight import attend_tight
from test_gpu_attend import Batch

pkg = load_pkg()
pytestmark = pytest.mark.gpu


def check(b, y, request=0, skip=(), **kw):
    t = sum(b.rows[:request])
    n, r = b.lengths[request], b.rows[request]
    pos = torch.arange(n - r, n, device="cuda")
    want, tol = attend_tight(b.q[t:t + r], values64(b.k[request]), values64(b.v[request]), pos, b.D ** -0.5,
                             split=b.q.dtype == torch.float16 and r * (b.Hq // b.H) <= 8, **kw)
    keep = [i for i in range(r) if i not in skip]
    close(y[t:t + r][keep], want[keep], tol[keep])


def store(b):
    b.cache.write(torch.cat(b.k), torch.cat(b.v), b.slots)


@pytest.mark.parametrize("D,Hq,H", [(64, 2, 1), (128, 4, 2), (256, 8, 2)])
@pytest.mark.parametrize("rows", (2, 4, 40, 130))
@pytest.mark.parametrize("size", (8, 16, 20, 30, 60, 100))
def test_a_value_that_a_row_does_not_see_leaves_it_alone(size, rows, D, Hq, H):
    b = Batch([300, 20], [rows, 1], Hq, H, D, 16, seed=size)
    b.v[0][299] *= 2.0 ** size                  # the last token: only the last row sees it
    store(b)
    y = b.run()
    check(b, y)
    check(b, y, 1)


@pytest.mark.parametrize("D,Hq,H", [(64, 2, 1), (128, 4, 2), (256, 8, 2)])
@pytest.mark.parametrize("rows", (4, 130))
def test_a_value_behind_a_window_leaves_rows_alone(rows, D, Hq, H):
    for size in (16, 24, 60):
        b = Batch([400], [rows], Hq, H, D, 16, seed=size)
        b.v[0][:400 - rows - 99] *= 2.0 ** size     # the first row sees one of them, the second none
        store(b)
        check(b, b.run(window=100), window=100)


@pytest.mark.parametrize("D,Hq,H", [(64, 2, 1), (128, 4, 2), (256, 8, 2)])
def test_large_values_of_no_weight(D, Hq, H):
    # a token that every row sees and whose weight is next to nothing
    for rows, sizes in ((1, (8, 16, 24, 40, 60)), (3, (16, 40)), (60, (8, 16, 20, 24, 40, 100))):
        for size in sizes:
            b = Batch([300], [rows], Hq, H, D, 16, seed=size)
            b.q.copy_(b.q.abs() + 0.5)
            b.k[0][50] = -64.0                  # scores of about -64 sqrt(D): weights of e^-500
            b.k[0][50, :, 0] = -60.0
            b.v[0][50] *= 2.0 ** size
            store(b)
            check(b, b.run())


@pytest.mark.parametrize("rows", (1, 4, 60))
def test_large_and_small_values(rows):
    for size in (-112, -106, -100, -80, -60, 60, 100, 116):
        b = Batch([300, 64], [rows, 1], 4, 2, 128, 16, seed=size & 255)
        b.v = [x * 2.0 ** size for x in b.v]
        store(b)
        y = b.run()
        assert y.isfinite().all()
        check(b, y)
        check(b, y, 1)
    b = Batch([300], [rows], 4, 2, 128, 16)
    b.v[0][...] = 3.0                           # no range at all
    b.v[0][17:40] = 2.0 ** 90
    b.v[0][250:] = 0
    store(b)
    check(b, b.run())


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("D,G", [(64, 1), (128, 4), (256, 2), (128, 12)])
@pytest.mark.parametrize("L", (16, 96, 640))
def test_light_weights_beside_heavy_ones(L, D, G, dtype):
    # one token in 16 weighs 2^10 to 2^14 times the others and has nothing but zeros: the result is the others' sum.
    # Scores are multiples of one number, exact up to its rounding, so that little is lost on the way to the second product
    g = torch.Generator().manual_seed(L + D)
    k, v = torch.full((L, 1, D), 7.0), torch.randint(-7, 9, (L, 1, D), generator=g).float()
    k[..., 0], k[..., 1], k[..., 2] = 0, 15, torch.randint(0, 4, (L, 1), generator=g).float()
    heavy = torch.arange(L) % 16 == torch.randint(0, 16, (1,), generator=g)
    k[heavy, :, 2], v[heavy] = 15, 0
    v[..., 0], v[..., 1] = -7, 8                              # every row: a step of 1, zero at code 7
    q = torch.zeros(1, G, D)
    q[..., 2] = 1
    cache = pkg.kvcache.KVCache4(-(-L // 16), 1, D, page_size=16, dtype=dtype)
    cache.write(k.to(dtype).cuda(), v.to(dtype).cuda(), torch.arange(L, dtype=torch.int32, device="cuda"))
    table = torch.arange(cache.n_pages, dtype=torch.int32, device="cuda")[None]
    y = cache.attend(q.to(dtype).cuda(), table, torch.tensor([L], dtype=torch.int32, device="cuda"), scale=0.9 * math.log(2)).double().cpu()
    p = torch.softmax(k[:, 0, 2].double() * 0.9 * math.log(2), 0)
    want = (p @ v[:, 0].double()).expand(1, G, D)
    # in steps: each product off by 2^-24 of 15 heavy weights (fp16: codes are normal numbers) or by 2^-16 of a heavy
    # weight (codes of four bits, two above the lowest), 16 a group; fp32 sums of at most 15, one a group and 40 at the ends.
    # bf16: the weights' own rounding, 2^-11 of half a step for the heavy ones and of 7.5 for what the others weigh (2^-6)
    drop = 16 * (15 * 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -16)
    if dtype == torch.bfloat16:
        drop += 2.0 ** -11 * (0.5 + 7.5 * 2.0 ** -6)
    tol = drop + 15 * (L / 16 + 40) * 2.0 ** -24 + 15 * 2.0 ** -22 + torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -25
    close(y[..., 2:], want[..., 2:], tol[..., 2:])
