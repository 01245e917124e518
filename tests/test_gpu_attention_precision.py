"""What a row's result may depend on, and how closely: attention on the GPU against bounds from the row's own weights."""
from __future__ import annotations

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
    for size in (-100, -80, -60, 60, 100, 116):
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
