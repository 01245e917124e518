"""Attention over the 4-bit cache on the GPU against the definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import load_pkg
from helpers_attention import attend64, close, values64

pkg = load_pkg()
kv = pkg.kvcache
pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")


class Batch:
    """Requests with lengths and new rows, their keys and values in pages in no order among pages of garbage
    (infinities and NaN included, in the parts of a page behind a request's last token too)."""

    def __init__(self, lengths, rows, Hq, H, D, page, dtype=torch.bfloat16, seed=0, gate=False, spare=2):
        self.lengths, self.rows, self.page, self.H, self.Hq, self.D = lengths, rows, page, H, Hq, D
        g = torch.Generator(device="cuda").manual_seed(seed + D + Hq + sum(lengths))
        counts = [-(-n // page) for n in lengths]
        n_pages = sum(counts) + spare
        self.cache = kv.KVCache4(n_pages, H, D, page_size=page, dtype=dtype)
        noise = torch.randint(0, 256, self.cache.k_codes.shape, dtype=torch.uint8, device="cuda", generator=g)
        for codes, pairs in ((self.cache.k_codes, self.cache.k_pairs), (self.cache.v_codes, self.cache.v_pairs)):
            codes.copy_(noise)
            pairs.fill_(math.nan)
            pairs[..., ::3, 1] = math.inf
            pairs[..., ::2, 0] = -3e4
        order = torch.randperm(n_pages, device="cuda", generator=g).int()
        width = max(counts + [1]) + 1
        self.table = torch.full((len(lengths), width), -1, **INT)
        self.k, self.v, at, slots = [], [], 0, []
        for b, n in enumerate(lengths):
            own = order[at:at + counts[b]]
            self.table[b, :counts[b]] = own
            at += counts[b]
            slots.append((own.long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:n].int())
            self.k.append((torch.randn(n, H, D, device="cuda", generator=g)
                           + torch.randn(H, D, device="cuda", generator=g)).to(dtype))
            self.v.append((torch.randn(n, H, D, device="cuda", generator=g) * (1 + torch.rand(n, H, 1, device="cuda", generator=g))
                           + torch.randn(H, 1, device="cuda", generator=g)).to(dtype))
        self.slots = torch.cat(slots)
        self.cache.write(torch.cat(self.k), torch.cat(self.v), self.slots)
        T = sum(rows)
        self.q = (1.5 * torch.randn(T, Hq, D, device="cuda", generator=g)).to(dtype)
        self.gate = torch.randn(T, Hq, D, device="cuda", generator=g).to(dtype) if gate else None
        self.kv_len = torch.tensor(lengths, **INT)
        self.row_start = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], **INT)

    def run(self, **kw):
        if "row_start" not in kw and any(r != 1 for r in self.rows):
            kw["row_start"] = self.row_start
        return self.cache.attend(kw.pop("q", self.q), self.table, self.kv_len, gate=self.gate, **kw)

    def check(self, y=None, scale=None, window=0, sinks=0, **kw):
        y = self.run(scale=scale, window=window, sinks=sinks, **kw) if y is None else y
        t = 0
        for b, (n, r) in enumerate(zip(self.lengths, self.rows)):
            pos = torch.arange(n - r, n, device="cuda")
            want, tol = attend64(self.q[t:t + r], values64(self.k[b]), values64(self.v[b]), pos,
                                 self.D ** -0.5 if scale is None else scale, window, sinks,
                                 None if self.gate is None else self.gate[t:t + r])
            close(y[t:t + r], want, tol, f"request {b}")
            t += r
        assert pkg._lib.lib().b200lut_device_status() == 0
        return y


SINGLE = [[1], [15], [16], [17], [1, 2, 3, 64], [255, 1, 100, 33, 16], [1000], [4099, 1, 700]]


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("Hq,H,D,page", [(1, 1, 64, 16), (6, 2, 64, 64), (4, 4, 128, 16), (8, 1, 128, 32), (3, 1, 256, 256),
                                         (16, 4, 256, 64), (16, 1, 128, 64), (12, 1, 256, 16), (40, 2, 64, 32), (64, 1, 128, 16)])
def test_single_rows(Hq, H, D, page, dtype):
    for i, lengths in enumerate(SINGLE):
        Batch(lengths, [1] * len(lengths), Hq, H, D, page, dtype, seed=i).check()


CHUNKS = [([5], [5]), ([40], [3]), ([70, 9, 200], [70, 1, 33]), ([300, 0, 17], [2, 0, 17]), ([513, 1025], [129, 1]),
          ([1200], [600])]


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("Hq,H,D,page", [(1, 1, 64, 16), (6, 2, 64, 128), (8, 8, 128, 16), (8, 1, 128, 32), (3, 1, 256, 64),
                                         (16, 4, 256, 16), (10, 2, 256, 256), (17, 1, 64, 16)])
def test_chunks_of_rows(Hq, H, D, page, dtype):
    for i, (lengths, rows) in enumerate(CHUNKS):
        Batch(lengths, rows, Hq, H, D, page, dtype, seed=i, gate=i % 2 == 1).check()


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 0), (16, 1), (100, 4), (37, 300), (4096, 4), (1, 1), (64, 15), (65, 17)])
@pytest.mark.parametrize("Hq,H,D,page", [(4, 1, 128, 16), (2, 2, 64, 64), (8, 2, 256, 32)])
def test_window_and_sinks(window, sinks, Hq, H, D, page):
    Batch([1, 33, 512, 1300], [1] * 4, Hq, H, D, page, seed=window).check(window=window, sinks=sinks)
    Batch([40, 333, 700], [40, 150, 3], Hq, H, D, page, torch.float16, seed=window, gate=True).check(window=window, sinks=sinks)


def test_long_rows_split_over_many_blocks():
    for dtype, Hq, H, D in ((torch.bfloat16, 16, 4, 256), (torch.float16, 8, 1, 128), (torch.bfloat16, 2, 2, 64)):
        b = Batch([70_001], [1], Hq, H, D, 64, dtype, gate=True)
        y = b.check()
        assert torch.equal(y, b.run())                                  # the order of the sums is fixed
        Batch([40_000, 3, 17_000], [2, 1, 64], Hq, H, D, 64, dtype).check()


def test_scale_and_peaked_rows():
    # one key towers over the others: p of the rest underflows, and the maximum moves along the row
    b = Batch([900, 50], [1, 1], 4, 1, 128, 16)
    b.check(scale=2.0)
    b.check(scale=0.0)                           # every token alike
    b.check(scale=-0.3)
    k = torch.linspace(-1, 1, 900, device="cuda")[:, None, None] * b.q[0, :1].float() / 4
    b.k[0] = (k + 0.01 * torch.randn_like(k)).bfloat16()
    b.cache.write(torch.cat(b.k), torch.cat(b.v), b.slots)
    b.check(scale=1.0)
    b.q.zero_()
    b.check()


def test_values_of_very_different_sizes():
    # the power of two in front of p * step follows the largest step so far
    for dtype in (torch.bfloat16, torch.float16):
        b = Batch([600, 333], [1, 3], 4, 2, 128, 32, dtype)
        top = 3e4 if dtype == torch.float16 else 1e30
        size = torch.logspace(-3, math.log10(top), 600, device="cuda")
        b.v[0] = (size[:, None, None] * torch.randn(600, 2, 128, device="cuda").clamp(-2, 2)).to(dtype)
        b.v[1] = (size.flip(0)[:333, None, None] * torch.randn(333, 2, 128, device="cuda").clamp(-2, 2)).to(dtype)
        b.cache.write(torch.cat(b.k), torch.cat(b.v), b.slots)
        b.check()


def test_queries_of_extreme_sizes():
    b = Batch([200], [4], 4, 1, 128, 16)
    b.q[0] *= 2.0 ** 60
    b.q[1] *= 2.0 ** -100
    b.q[2, 0, 1:] = 0
    b.check(scale=2.0 ** -70)
    b.q[0] = 1
    b.q[3, 2, 5] = math.nan
    y = b.run()
    assert y[3, 2].isnan().all() and not y[3, 1].isnan().any() and not y[:3].isnan().any()


def test_poisoned_rows_are_seen_where_they_are_visible():
    for rows in ([1, 1], [8, 1]):
        b = Batch([100, 60], rows, 8, 2, 64, 16, seed=5)
        b.k[0][95, 1, 3] = math.nan
        b.v[1][20, 0, 9] = math.inf
        b.cache.write(torch.cat(b.k), torch.cat(b.v), b.slots)
        y = b.check()
        first = rows[0]
        # rows at positions before 95 do not see the key
        want = torch.zeros(sum(rows), 8, dtype=torch.bool, device="cuda")
        want[max(0, 95 - (100 - first)):first, 4:] = True
        want[first:, :4] = True
        assert torch.equal(y.isnan().all(-1), want) and torch.equal(y.isnan().any(-1), want)


def test_rows_that_see_nothing_and_rows_of_no_request():
    b = Batch([40, 0, 3], [1, 1, 1], 4, 2, 128, 16)
    y = b.run()
    assert not y[1].any() and y[0].any()
    # more rows than tokens: the first ones lie before the sequence; the buffer is longer than the batch
    for D, G in ((128, 2), (256, 4)):
        b = Batch([5, 20], [9, 2], 2 * G, 2, D, 16)
        q = torch.cat((b.q, torch.full((7, 2 * G, D), math.nan, device="cuda", dtype=b.q.dtype)))
        out = torch.full_like(q, 7.0)
        assert b.run(q=q, out=out) is out
        assert not out[:4].any() and (out[11:] == 7).all()
        b.check(out[:11])
        out = torch.full_like(q, 7.0)
        b.cache.attend(q, b.table, torch.zeros(2, **INT), b.row_start, out=out)
        assert not out[:11].any() and (out[11:] == 7).all()


def test_lengths_and_starts_beyond_their_buffers():
    b = Batch([64, 30], [1, 1], 2, 1, 64, 16)
    want = b.run()
    # a length beyond the row of the table ends with it; there the table's pages are -1: hidden, and reported
    y = b.cache.attend(b.q, b.table, torch.tensor([64, 10 ** 9], **INT))
    assert pkg._lib.lib().b200lut_device_status() == 0x6200
    assert torch.equal(y[0], want[0])
    # starts beyond the rows, or running backwards, name no row
    for start in ([0, 1, 9], [0, 2 ** 31 - 1, 2 ** 31 - 1], [-5, 1, 0], [2, 1, 0]):
        out = torch.full_like(b.q, 3.0)
        b.cache.attend(b.q, b.table, b.kv_len, torch.tensor(start, **INT), out=out)
    assert pkg._lib.lib().b200lut_device_status() == 0


def test_pages_outside_the_cache_are_hidden_and_reported():
    for rows in ([1], [20]):
        b = Batch([80], rows, 8, 2, 128, 16)
        table = b.table.clone()
        for bad in (-1, b.cache.n_pages, 2 ** 31 - 1, -2 ** 31):
            b.table = table.clone()
            b.table[0, 2] = bad
            y = b.run()
            assert pkg._lib.lib().b200lut_device_status() == 0x6200
            keep = [i for i in range(80) if not 32 <= i < 48]
            pos = torch.arange(80 - rows[0], 80, device="cuda")
            seen = torch.where(pos >= 48, pos - 16, pos.clamp(max=31))
            want, tol = attend64(b.q, values64(b.k[0][keep]), values64(b.v[0][keep]), seen, 128 ** -0.5)
            close(y, want, tol, str(bad))


def test_offsets_beyond_32_bits():
    H, D, page, L = 4, 256, 64, 1000
    far, near = pkg.kvcache.KVCache4(150000, H, D, page_size=page), pkg.kvcache.KVCache4(16, H, D, page_size=page)
    assert far.k_codes.numel() > 2 ** 32
    pages = torch.arange(16, **INT)
    slots = (pages.long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:L].int()
    k, v = (torch.randn(L, H, D, device="cuda").bfloat16() for _ in range(2))
    far.write(k, v, slots + (150000 - 16) * page)
    near.write(k, v, slots)
    for rows in (1, 70):
        q, start, n = torch.randn(rows, 2 * H, D, device="cuda").bfloat16(), torch.tensor([0, rows], **INT), torch.tensor([L], **INT)
        assert torch.equal(far.attend(q, pages[None] + (150000 - 16), n, start), near.attend(q, pages[None], n, start))


def test_strides():
    b = Batch([100, 37, 5], [1, 20, 5], 8, 2, 128, 32, gate=True)
    want = b.check()
    T = b.q.shape[0]
    wide = torch.randn(T, 8, 3 * 128, device="cuda").bfloat16()
    wide[..., :128], wide[..., 128:256] = b.q, b.gate
    b.q, b.gate, out = wide[..., :128], wide[..., 128:256], torch.empty(T + 1, 8, 136, device="cuda", dtype=torch.bfloat16)
    table = torch.full((3, 40), -1, **INT)
    table[:, 3:3 + b.table.shape[1]] = b.table
    b.table = table[:, 3:3 + b.table.shape[1]]
    assert torch.equal(b.run(), want)
    assert torch.equal(b.run(out=out[1:, :, :128]), want)
    b.q = torch.randn(T, 8, 129, device="cuda").bfloat16()[..., 1:].copy_(b.q)       # not 16-byte rows: copied
    assert torch.equal(b.run(), want)
    b.q = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(b.run(), want)
    b.table = b.table.T.contiguous().T
    assert torch.equal(b.run(), want)


def test_captured_with_lengths_that_grow():
    b = Batch([100, 37, 500], [1, 1, 1], 8, 2, 128, 16, gate=True)
    c = Batch([60, 90], [30, 1], 8, 2, 128, 16)
    graphs, outs = [], []
    for x in (b, c):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(x.run())
    for step in range(3):
        for x in (b, c):
            x.lengths = [n - 7 for n in x.lengths]
            x.kv_len.copy_(torch.tensor(x.lengths, **INT))
            x.k, x.v = [t[:n] for t, n in zip(x.k, x.lengths)], [t[:n] for t, n in zip(x.v, x.lengths)]
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        b.check(outs[0])
        c.check(outs[1])


def test_two_streams_at_once():
    batches = [Batch([3000 + 100 * i, 50], [1, 1 + 30 * (i % 2)], 8, 2, 128, 16, seed=i) for i in range(4)]
    want = [b.check() for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = [[] for _ in batches]
    for _ in range(5):
        for b, s, g in zip(batches, streams, got):
            with torch.cuda.stream(s):
                g.append(b.run())
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for g, w in zip(got, want) for y in g)


def test_many_requests():
    g = torch.Generator().manual_seed(4)
    lengths = torch.randint(0, 60, (700,), generator=g).tolist()
    b = Batch(lengths, [1] * 700, 2, 1, 64, 16)
    y = b.run()
    for i in range(0, 700, 41):
        n = lengths[i]
        want, tol = attend64(b.q[i:i + 1], values64(b.k[i]), values64(b.v[i]), torch.tensor([n - 1], device="cuda"), 0.125)
        close(y[i:i + 1], want, tol, f"request {i}")
    rows = [min(n, 1 + i % 5) for i, n in enumerate(lengths)]
    b = Batch(lengths, rows, 4, 1, 64, 16)
    b.check()
