"""The attention side at the ends of what its arguments can say, on the GPU."""
from __future__ import annotations

import pytest
import torch

from conftest import load_pkg
from helpers_attention import attend64, close, values64
from test_gpu_attend import Batch

pkg = load_pkg()
kv = pkg.kvcache
pytestmark = pytest.mark.gpu
INT = dict(dtype=torch.int32, device="cuda")


def status():
    return pkg._lib.lib().b200lut_device_status()


def test_plan_of_requests_that_would_pass_the_largest_length():
    # a row of the table that reaches beyond 2^31 tokens: the length stops before
    width, page = 2 ** 23 + 1, 256
    table = torch.full((2, width), 3, **INT)
    last = 2 ** 31 - 1
    for fresh, served in ((5, True), (6, False), (300, False), (2 ** 31 - 1, False)):
        step = kv.plan_step(torch.tensor([2, last - 5], **INT), torch.tensor([1, fresh], **INT), table,
                            torch.arange(9, **INT), torch.zeros(1, **INT), page, 320)
        assert step.served.tolist() == [True, served]
        assert step.kv_len.tolist() == [3, last if served else last - 5] and step.taken.item() == 0
        rows = 5 if served else 0
        want = [3 * page + (last - 5 + i) % page for i in range(rows)] + [-1] * (319 - rows)
        assert step.slots.tolist() == [3 * page + 2] + want
        assert step.positions.min().item() >= 0
    assert (table == 3).all()


@pytest.mark.parametrize("rows", (1, 30))
def test_windows_and_sinks_beyond_32_bits(rows):
    b = Batch([500], [rows], 4, 2, 128, 16)
    want = b.check()
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 100, 2 ** 70):
        assert torch.equal(b.run(window=window), want), window
        assert torch.equal(b.run(window=window, sinks=window), want), window
    few = b.check(window=100)
    assert not torch.equal(few, want)
    every = b.check(window=100, sinks=500)
    for sinks in (2 ** 31, 2 ** 32, 2 ** 32 + 3, 2 ** 70):             # every token is among the first so many
        assert torch.equal(b.run(window=100, sinks=sinks), every), sinks


@pytest.mark.parametrize("lengths,rows", [([5, 20], [9, 2]), ([2, 40], [3, 1]), ([0, 7], [1, 30])])
def test_windows_near_two_to_the_31_with_rows_before_the_sequence(lengths, rows):
    for D, Hq, H in ((128, 4, 2), (64, 2, 1), (256, 16, 1)):
        b = Batch(lengths, rows, Hq, H, D, 16)
        want = b.run()
        assert want.any()
        for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 9, 2 ** 30):
            assert torch.equal(b.run(window=window), want), window
            assert torch.equal(b.run(window=window, sinks=3), want), window
    assert status() == 0


@pytest.mark.parametrize("rows", (1, 2, 60))
def test_the_longest_sequences(rows):
    # a table of 2^23 pages of 256 tokens that names eight pages over and over; windows keep what is read short
    H, D, page, window = 1, 64, 256, 700
    cache = kv.KVCache4(8, H, D, page_size=page)
    g = torch.Generator(device="cuda").manual_seed(rows)
    k, v = (torch.randn(8 * page, H, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    cache.write(k, v, torch.arange(8 * page, **INT))
    table = (torch.arange(2 ** 23, **INT) % 8)[None]
    q = torch.randn(rows, 2, D, device="cuda", generator=g).bfloat16()
    start = torch.tensor([0, rows], **INT)
    for short in (1, 2, 17, 130, 300):
        n = 2 ** 31 - short
        y = cache.attend(q, table, torch.tensor([n], **INT), None if rows == 1 else start, window=window)
        # the last tokens as they lie in a short sequence: 2^31 is a multiple of what the table repeats
        lies = torch.arange(8 * page - short - rows - window, 8 * page - short, device="cuda")
        pos = torch.arange(window, window + rows, device="cuda")
        want, tol = attend64(q, values64(k[lies]), values64(v[lies]), pos, D ** -0.5, window)
        close(y, want, tol, str(short))
    assert status() == 0


@pytest.mark.parametrize("D,Hq,H", [(64, 2, 1), (128, 4, 1), (256, 8, 2)])
@pytest.mark.parametrize("rows", (1, 40))
def test_queries_up_to_the_largest(rows, D, Hq, H):
    # queries of up to 2^127 over keys so small that the scores are ordinary
    for e in (63, 64, 110, 117, 119, 121, 124, 126):
        b = Batch([200, 30], [rows, 1], Hq, H, D, 16, seed=e)
        b.q[0] = (b.q[0].float().clamp(-1.99, 1.99) * 2.0 ** e).bfloat16()
        b.q[-1] = b.q[-1].abs().clamp(0.5, 1.99)                       # their plain sum passes what fp32 holds
        b.q[-1] = (b.q[-1].float() * 2.0 ** 126).bfloat16()
        b.k[0] = (b.k[0].float() * 2.0 ** -e).bfloat16()
        b.k[1] = (b.k[1].float() * 2.0 ** -126).bfloat16()
        b.cache.write(torch.cat(b.k), torch.cat(b.v), b.slots)
        y = b.check()
        assert y.isfinite().all()
        b.check(scale=-0.3)


def test_single_tokens_and_heads_in_rows_of_odd_strides():
    bf = torch.bfloat16
    rot = pkg.rotary.AxisRotary(64, theta=1e4)
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(5, 4 * 128 + 1 * 128 + 3, device="cuda", generator=g).to(bf)
    q, k = wide[:, :512].unflatten(1, (4, 128))[:1], wide[:, 512:640].unflatten(1, (1, 128))[:1]
    assert q.stride(0) % 8 and k.stride(0) % 8 and q.is_contiguous()
    pos = torch.tensor([77], device="cuda")
    for _ in range(2):                                  # with and without the rotation's tables in place
        assert all(torch.equal(a, b) for a, b in zip(rot(q, k, pos), rot(q.clone(memory_format=torch.contiguous_format).reshape(1, 4, 128),
                                                                         torch.empty_like(k).copy_(k), pos)))
    cache, plain = (kv.KVCache4(2, 1, 128, page_size=16) for _ in range(2))
    slot = torch.tensor([5], **INT)
    cache.write(k, k, slot)
    dense = torch.empty(1, 1, 128, device="cuda", dtype=bf).copy_(k)
    plain.write(dense, dense, slot)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(slot), plain.read(slot))) and cache.read(slot)[0].any()
    table, n = torch.tensor([[0]], **INT), torch.tensor([6], **INT)
    dense = torch.empty(1, 4, 128, device="cuda", dtype=bf).copy_(q)
    want = plain.attend(dense, table, n, gate=dense)
    out = torch.zeros(2, 4 * 128 + 1, device="cuda", dtype=bf)
    to = out[:, :512].unflatten(1, (4, 128))[:1]
    assert to.stride(0) % 8
    assert torch.equal(cache.attend(q, table, n, gate=q), want)
    assert cache.attend(q, table, n, gate=q, out=to) is to and torch.equal(to, want) and not out[1].any() and not out[0, 512]
    odd = torch.zeros(2 * 513, device="cuda", dtype=bf)[1:].as_strided((1, 4, 128), (513, 128, 1))
    with pytest.raises(ValueError, match="16-byte"):
        cache.attend(q, table, n, out=odd)
    # one head, odd strides between tokens' heads
    one = torch.randn(3, 2, 136, device="cuda", generator=g).to(bf)[:, :1, :128]
    cache.write(one, one, torch.arange(3, **INT))
    assert cache.read(torch.arange(3, **INT))[0].any()


@pytest.mark.parametrize("rows", (1, 40))
def test_a_bad_slot_does_not_hide_a_bad_page(rows):
    b = Batch([80], [rows], 8, 2, 128, 16)
    assert status() == 0
    b.cache.write(b.k[0][:2], b.v[0][:2], torch.tensor([-1, b.cache.n_pages * 16], **INT))
    b.table[0, 1] = b.cache.n_pages
    b.run()
    assert [status() for _ in range(3)] == [0x6100, 0x6200, 0]
    two = Batch([80, 300], [1, 40], 8, 2, 128, 16)          # both kernels of one call: one word
    two.table[:, 1] = -1
    two.run()
    assert [status() for _ in range(2)] == [0x6200, 0]


@pytest.mark.parametrize("Hq,H,D,page", [(4, 2, 64, 16), (8, 2, 128, 16), (8, 2, 256, 32), (2, 1, 128, 64)])
@pytest.mark.parametrize("rows", (1, 3, 50))
def test_pages_that_no_row_sees_may_be_given_away(rows, Hq, H, D, page):
    for n in (500, 507, 511, 530):
        for window, sinks in ((20, 0), (33, 4), (100, 70)):
            b = Batch([n, 40], [rows, 1], Hq, H, D, page, seed=n)
            want = b.run(window=window, sinks=sinks)
            assert status() == 0
            kept = -(-sinks // page)
            b.table[0, kept:(n - rows - window + 1) // page] = -1
            assert torch.equal(b.run(window=window, sinks=sinks), want)
            assert status() == 0
            b.table[0, (n - rows - window + 1) // page] = -1            # the first row sees a token of it
            b.run(window=window, sinks=sinks)
            assert status() == 0x6200 and status() == 0


def test_scales_that_32_bits_do_not_hold():
    b = Batch([40], [1], 4, 2, 128, 16)
    for scale in (1e300, -1e39, 2.0 ** 127, float("inf")):
        with pytest.raises(ValueError, match="scale"):
            b.run(scale=scale)
    b.q.mul_(2.0 ** -100)
    b.check(scale=2.0 ** 96)


@pytest.mark.parametrize("D,R", [(64, 32), (128, 128), (256, 64)])
def test_norm_of_heads_whose_squares_pass_32_bits(D, R):
    from helpers_attention import rotate64
    rot = pkg.rotary.AxisRotary(R, theta=1e4)
    g = torch.Generator(device="cuda").manual_seed(D)
    for T in (1, 9, 3000):
        q, k = (torch.randn(T, n, D, device="cuda", generator=g) for n in (5, 2))
        size = torch.randint(55, 125, (T, 5, 1), device="cuda", generator=g)
        q = (q * torch.where(size % 3 == 0, 0, size).float().exp2()).bfloat16()
        k = (k * 2.0 ** 62).bfloat16()
        gains = [(1 + 0.1 * torch.randn(D, device="cuda", generator=g)).bfloat16() for _ in range(2)]
        pos = torch.arange(T, device="cuda")
        for x, y, gain in zip((q, k), rot(q, k, pos, *gains), gains):
            want, tol = rotate64(x, pos[None], R, 1e4, rot.axis, gain)
            close(y, want, tol)
    q = torch.zeros(1, 1, D, device="cuda", dtype=torch.bfloat16)
    q[0, 0, R - 1] = float("inf")                           # 0 times infinity stays NaN, the others are zero
    y = rot(q, k[:1], pos[:1], *gains)[0]
    assert y.isnan().any() and (y.isnan() | (y == 0)).all()


def test_sizes_that_32_bits_do_not_hold():
    i = torch.zeros(3, **INT)
    for room in (2 ** 31, 2 ** 32 + 8, 2 ** 64):
        with pytest.raises(ValueError, match="2\\^31"):
            kv.plan_step(i, i, torch.zeros(3, 2, **INT), i, i[:1], page_size=16, max_tokens=room)
    wide = i[:1].expand(1, 2 ** 32 + 1)                     # one element, read as so many
    with pytest.raises(ValueError, match="2\\^31"):
        kv.plan_step(i[:1], i[:1], torch.zeros(1, 2, **INT), wide[0], i[:1], page_size=16, max_tokens=8)
    cache = kv.KVCache4(2, 1, 64, page_size=16)
    with pytest.raises(ValueError, match="2\\^31"):
        cache.attend(torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16), wide, i[:1])


@pytest.mark.parametrize("Hq,H,D", [(8, 2, 128), (24, 2, 64), (16, 4, 256)])
def test_the_result_in_the_place_of_the_queries_or_gates(Hq, H, D):
    for lengths, rows in (([9000, 40, 700], [1, 1, 1]), ([5000, 300, 20], [200, 1, 9])):
        b = Batch(lengths, rows, Hq, H, D, 32, gate=True)
        want, q, gate = b.run(), b.q.clone(), b.gate.clone()
        for _ in range(3):
            b.q = q.clone()
            assert b.run(out=b.q) is b.q and torch.equal(b.q, want)
            b.q, b.gate = q, gate.clone()
            assert b.run(out=b.gate) is b.gate and torch.equal(b.gate, want)
            b.gate = gate


def test_one_table_for_every_request_and_lengths_with_strides():
    b = Batch([300], [1], 8, 2, 128, 16)
    q = b.q.expand(5, 8, 128)                                   # one query, five lengths
    lengths = torch.tensor([[300, 0], [17, 0], [0, 0], [1, 0], [255, 0]], **INT)[:, 0]
    y = b.cache.attend(q, b.table.expand(5, -1), lengths)
    for i, n in enumerate(lengths.tolist()):
        want, tol = attend64(b.q, values64(b.k[0][:n]), values64(b.v[0][:n]), torch.tensor([n - 1], device="cuda"), 128 ** -0.5)
        close(y[i:i + 1], want, tol, str(n))
    assert status() == 0
