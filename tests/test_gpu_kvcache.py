"""The step plan and the 4-bit cache on the GPU: integers exactly, rows against the definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import load_pkg
from helpers_attention import close, floor, unit, values64

pkg = load_pkg()
kv = pkg.kvcache
pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- step plan

def plan_by_hand(cached, fresh, table, free, taken, page, room):
    """The definition, request by request."""
    table = [list(r) for r in table]
    start, total, upto, used = [], 0, taken, taken
    kv_len, served, pos, slots = [], [], [0] * room, [-1] * room
    for b, (c, n) in enumerate(zip(cached, fresh)):
        c, n = max(c, 0), max(n, 0)
        have, want = -(-c // page), -(-(c + n) // page)
        start.append(min(total, room))
        fits = want <= len(table[b]) and total + n <= room
        need = want - have if fits else 0
        upto += need
        ok = fits and (need == 0 or upto <= len(free))
        if ok:
            for j in range(need):
                table[b][have + j] = free[upto - need + j]
            if need:
                used = upto
        for i in range(n):
            if total + i < room:
                pos[total + i] = c + i
                entry = table[b][(c + i) // page] if ok else -1
                slots[total + i] = entry * page + (c + i) % page if entry >= 0 else -1
        total += n
        kv_len.append(c + n if ok else c)
        served.append(ok)
    start.append(min(total, room))
    return start, kv_len, pos, slots, used, served, table


def plan_case(cached, fresh, table, free, taken, page, room):
    dev = dict(dtype=torch.int32, device="cuda")
    t = torch.tensor(table, **dev)
    args = (torch.tensor(cached, **dev), torch.tensor(fresh, **dev), t, torch.tensor(free, **dev),
            torch.tensor([taken], **dev))
    p = kv.plan_step(*args, page_size=page, max_tokens=room)
    want = plan_by_hand(cached, fresh, table, free, taken, page, room)
    got = [p.row_start.tolist(), p.kv_len.tolist(), p.positions.tolist(), p.slots.tolist(), p.taken.item(),
           p.served.tolist(), t.tolist()]
    for name, g, w in zip(("row_start", "kv_len", "positions", "slots", "taken", "served", "block_table"), got, want):
        assert g == w, name
    again = kv.plan_step(*args, page_size=page, max_tokens=room)
    assert all(torch.equal(a, b) for a, b in zip(p, again)) and t.tolist() == want[-1]
    return p


@pytest.mark.parametrize("B,longest,page,slack", [(1, 1, 16, 0), (1, 300, 64, 5), (8, 1, 64, 0), (31, 40, 16, 100),
                                                   (129, 7, 32, 3), (513, 20, 16, 0), (1500, 9, 16, 64), (2100, 1, 256, 0)])
def test_plan(B, longest, page, slack):
    g = torch.Generator().manual_seed(B)
    fresh = torch.randint(0 if B > 1 else 1, longest + 1, (B,), generator=g).tolist()
    cached = torch.randint(0, 5 * page, (B,), generator=g).tolist()
    width = max(-(-(c + n) // page) for c, n in zip(cached, fresh)) + 1
    pages = torch.randperm(20000, generator=g).tolist()
    table = [[-1] * width for _ in range(B)]
    for b, c in enumerate(cached):
        for j in range(-(-c // page)):
            table[b][j] = pages.pop()
    plan_case(cached, fresh, table, pages[:6000], 17, page, max(1, sum(fresh) + slack))


def test_plan_that_does_not_fit():
    table = [[7, -1, -1], [8, 9, -1], [-1, -1, -1], [3, 4, 5]]
    free = list(range(100, 104))
    # request 1 wants a fourth page of a row of three, request 3 too; the others are served
    plan_case([10, 40, 0, 48], [5, 20, 16, 1], table, free, 0, 16, 64)
    # the free list runs out at the second request; the one that needs no page is served, so is what follows it without
    plan_case([16, 16, 3, 20], [32, 33, 2, 3], table, free, 1, 16, 128)
    # rows that would end behind the buffers
    plan_case([0, 0, 5, 5], [10, 10, 3, 1], table, free, 0, 16, 12)
    # nothing left, nothing free
    plan_case([5, 5, 5, 5], [1, 1, 12, 0], table, free, 4, 16, 16)
    plan_case([5, 5, 0, 5], [1, 1, 1, 0], table, [], 0, 16, 16)
    # negative counts are zero, a negative page has no slots
    plan_case([-3, 16, 5, 5], [2, -1, 1, 4], [[-1, -1], [-1, -1], [-2, 6], [4, 4]], free, 0, 16, 16)
    plan_case([0], [0], [[-1]], free, 0, 16, 1)


def test_plan_of_many_requests_and_overflowing_counts():
    dev = dict(dtype=torch.int32, device="cuda")
    B = 8192
    big = torch.full((B,), 2 ** 30, **dev)                       # the sums pass 2^42
    table = torch.full((B, 3), -1, **dev)
    p = kv.plan_step(torch.zeros(B, **dev), big, table, torch.arange(10, **dev), torch.zeros(1, **dev), page_size=16,
                     max_tokens=100)
    assert not p.served.any() and (p.slots == -1).all() and (table == -1).all() and p.taken.item() == 0
    assert p.row_start.tolist() == [0] + [100] * B


def test_plan_of_pages_that_are_none():
    dev = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[3, 2 ** 31 - 1], [2 ** 27, -1], [-7, -1]], **dev)
    step = kv.plan_step(torch.tensor([17, 1, 2], **dev), torch.tensor([1, 2, 1], **dev), table, torch.arange(4, **dev),
                        torch.zeros(1, **dev), 16, 4)
    # slots of pages beyond every cache do not wrap into one: writes skip and report them; negative pages have no slot
    assert step.slots.tolist() == [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, -1]


def test_plan_captured_and_replayed():
    dev = dict(dtype=torch.int32, device="cuda")
    cached, fresh = torch.tensor([15, 31], **dev), torch.tensor([1, 1], **dev)
    table = torch.tensor([[0, -1, -1], [1, 2, -1]], **dev)
    free, taken = torch.arange(10, 20, **dev), torch.zeros(1, **dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = kv.plan_step(cached, fresh, table, free, taken, page_size=16, max_tokens=4)
        cached.copy_(p.kv_len)
        taken.copy_(p.taken)
    for _ in range(3):
        graph.replay()
    assert cached.tolist() == [18, 34] and taken.item() == 2 and table.tolist() == [[0, 10, -1], [1, 2, 11]]
    assert p.slots.tolist() == [10 * 16 + 1, 11 * 16 + 1, -1, -1]


# --------------------------------------------------------------------------- rows in and out

def bound(x, want):
    """One rounding to the type, and fp32 arithmetic on lo and the range: the step, the product and the sum are each
    off by less than 2^-23 of the larger of |lo| and the range."""
    size = x.double().abs().amax(-1, keepdim=True) + (x.double().amax(-1, keepdim=True) - x.double().amin(-1, keepdim=True))
    return unit(x.dtype) * want.abs() + 2.0 ** -21 * size + floor(x.dtype)


def round_trip(cache, k, v, slots):
    cache.write(k, v, slots)
    got = cache.read(slots)
    for name, x, y in zip("kv", (k, v), got):
        want = values64(x)
        close(y, want, bound(x, want), name)
    return got


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("D,H,page,T", [(64, 1, 16, 1), (64, 3, 32, 77), (128, 8, 16, 130), (128, 1, 256, 5),
                                        (256, 4, 64, 333), (256, 1, 128, 1)])
def test_rows_round_trip(D, H, page, T, dtype):
    g = torch.Generator(device="cuda").manual_seed(D + T)
    pages = -(-T // page) + 3
    cache = kv.KVCache4(pages, H, D, page_size=page, dtype=dtype)
    assert cache.nbytes == sum(t.numel() * t.element_size() for t in (cache.k_codes, cache.v_codes, cache.k_pairs, cache.v_pairs))
    k = (torch.randn(T, H, D, device="cuda", generator=g) + torch.randn(H, D, device="cuda", generator=g)).to(dtype)
    v = torch.randn(T, H, D, device="cuda", generator=g).to(dtype)
    for slots in (torch.arange(T), torch.randperm(pages * page)[:T], torch.arange(T) + page - 3):
        round_trip(cache, k, v, slots.int().cuda())


def test_documented_layout():
    """The codes and pairs lie where the header says."""
    D, H, page = 128, 2, 32
    cache = kv.KVCache4(3, H, D, page_size=page)
    k, v = torch.randn(40, H, D, device="cuda").bfloat16(), torch.randn(40, H, D, device="cuda").bfloat16()
    slots = torch.randperm(96)[:40].int().cuda()
    cache.write(k, v, slots)
    for x, codes, pairs, value in ((k, cache.k_codes, cache.k_pairs, False), (v, cache.v_codes, cache.v_pairs, True)):
        xd = x.double()
        lo, hi = xd.amin(-1), xd.amax(-1)
        want = torch.round(15 * (xd - lo[..., None]) / (hi - lo)[..., None]).long()
        page_i, off = (slots // page).long(), (slots % page).long()
        assert torch.equal(pairs[page_i, :, off].double(), torch.stack((lo, hi), -1))
        words = codes.view(torch.int32).long() & 0xFFFFFFFF                       # [pages, H, page * D / 8]
        w = torch.arange(D // 8, device="cuda")
        s = off[:, None] % 16
        at = off[:, None] * (D // 8) + w if not value else \
            ((off[:, None] // 16) * (D // 64) + w // 8) * 128 + ((s // 4) * 8 + w % 8) * 4 + s % 4
        for h in range(H):
            word = words[page_i[:, None], h, at]
            got = (word[..., None] >> (4 * torch.arange(8, device="cuda"))) & 15
            assert torch.equal(got.reshape(40, D), want[:, h])


def test_borders_and_constant_rows():
    # codes half way between two: 15 (x - lo) / (hi - lo) = n + 1/2 exactly, decided half to even
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.arange(64, dtype=torch.float32).fmod(31) / 2           # 0, 0.5 ... 15: range 15
        x[0], x[1] = 0, 15
        k = x.to(dtype).view(1, 1, 64).cuda()
        cache = kv.KVCache4(1, 1, 64, page_size=16, dtype=dtype)
        slots = torch.tensor([5], dtype=torch.int32, device="cuda")
        got = round_trip(cache, k, 3 * k, slots)
        assert torch.equal(got[0].double(), torch.round(k.double())) and torch.equal(got[1].double(), 3 * torch.round(k.double()))
        flat = torch.full((1, 1, 64), -1.75, dtype=dtype, device="cuda")
        assert all(torch.equal(t, flat) for t in round_trip(cache, flat, flat, slots))
        ends = torch.randn(1, 1, 64, device="cuda").to(dtype)            # the smallest and the largest come back exactly
        got = round_trip(cache, ends, ends, slots)[0]
        assert got.min() == ends.min() and got.max() == ends.max()


def test_quotients_next_to_a_border():
    # 15 (x - lo) of more than 24 bits: 6.50000004, which is 6.5 in fp32
    lo, hi, near = -2.177734375, 2.83984375, -0.0034503936767578125
    x = torch.full((4, 1, 64), lo, device="cuda", dtype=torch.float16)
    x[..., 1], x[:2, :, 5], x[2:, :, 7] = hi, near, near
    cache = kv.KVCache4(2, 1, 64, page_size=16, dtype=torch.float16)
    k, v = round_trip(cache, x, x.flip(-1), torch.arange(4, device="cuda").int())
    assert (k[0, 0, 5] > 0.16) and torch.equal(v, k.flip(-1))
    # bf16: a tiny element of a symmetric row, and a row with a tiny smallest element
    x = torch.full((4, 1, 64), -2.484375, device="cuda", dtype=torch.bfloat16)
    x[..., 1], x[:, 0, 5] = 2.484375, torch.tensor([-4.9e-8, 4.9e-8, 0.0, -1e-12])
    y = torch.full((4, 1, 64), 1e-6, device="cuda", dtype=torch.bfloat16)
    y[..., 1], y[..., 5], y[..., 6] = 30.0, 15.0, 1.0
    cache = kv.KVCache4(2, 1, 64, page_size=16)
    k, v = round_trip(cache, x, y, torch.arange(4, device="cuda").int())
    assert (k[:, 0, 5] > 0).tolist() == [False, True, True, False] and (v[:, 0, 6] < 0.1).all()


def test_extreme_rows():
    for dtype in (torch.bfloat16, torch.float16):
        info = torch.finfo(dtype)
        rows = torch.randn(6, 1, 128, device="cuda").to(dtype)
        rows[0, 0, 7] = math.nan
        rows[1, 0, 100] = math.inf
        rows[2, 0, 3] = -math.inf
        rows[3] = rows[3] * info.smallest_normal
        rows[4, 0, 0], rows[4, 0, 1] = info.max, -info.max        # bf16: a range beyond 2^120 reads NaN
        rows[5] = 0
        cache = kv.KVCache4(1, 1, 128, page_size=16, dtype=dtype)
        slots = torch.arange(6, dtype=torch.int32, device="cuda")
        cache.write(rows, rows, slots)
        k, v = cache.read(slots)
        assert k[:3].isnan().all() and v[:3].isnan().all()
        assert k[4].isnan().all() == (dtype == torch.bfloat16)
        assert not k[5].any()
        want = values64(rows[3:4])
        close(k[3:4], want, bound(rows[3:4], want), "subnormal rows")


def test_slots_that_are_skipped():
    cache = kv.KVCache4(2, 2, 64, page_size=16)
    k, v = torch.randn(4, 2, 64, device="cuda").bfloat16(), torch.randn(4, 2, 64, device="cuda").bfloat16()
    assert pkg._lib.lib().b200lut_device_status() == 0
    cache.write(k, v, torch.tensor([3, -1, 31, -7], dtype=torch.int32, device="cuda"))
    assert pkg._lib.lib().b200lut_device_status() == 0
    all_k, all_v = cache.read(torch.arange(32, dtype=torch.int32, device="cuda"))
    rest = [i for i in range(32) if i not in (3, 31)]
    assert not all_k[rest].any() and not all_v[rest].any() and all_k[3].any() and all_v[31].any()
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_pairs, cache.v_pairs)]
    cache.write(k[:2], v[:2], torch.tensor([32, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    assert pkg._lib.lib().b200lut_device_status() == 0x6100 and pkg._lib.lib().b200lut_device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k_codes, cache.v_codes, cache.k_pairs, cache.v_pairs)))
    got = cache.read(torch.tensor([32, -1, 3], dtype=torch.int32, device="cuda"))
    assert pkg._lib.lib().b200lut_device_status() == 0x6100
    assert not got[0][:2].any() and torch.equal(got[0][2], all_k[3])
    cache.write(k[:0], v[:0], torch.empty(0, dtype=torch.int32, device="cuda"))
    assert cache.read(torch.empty(0, dtype=torch.int32, device="cuda"))[0].shape == (0, 2, 64)


def test_strided_rows():
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = torch.randn(50, 4 * 128 + 4 * 128, device="cuda", generator=g).half()
    k, v = rows[:, :512].view(50, 4, 128), rows[:, 512:].view(50, 4, 128)
    cache = kv.KVCache4(8, 4, 128, page_size=16, dtype=torch.float16)
    wide = torch.arange(100, dtype=torch.int32, device="cuda").view(50, 2)
    round_trip(cache, k, v, wide[:, 1])
    round_trip(cache, k.transpose(0, 1).contiguous().transpose(0, 1), v.flip(0), wide[:, 0])
    odd = torch.randn(50, 4, 130, device="cuda", generator=g).half()[..., 1:129]
    round_trip(cache, odd, v, wide[:, 0])


def test_offsets_beyond_32_bits():
    # 4.8 GB of key codes: the last pages' offsets pass 2^32
    cache = kv.KVCache4(147_000, 1, 256, page_size=256)
    assert cache.k_codes.numel() > 2 ** 32
    k, v = torch.randn(300, 1, 256, device="cuda").bfloat16(), torch.randn(300, 1, 256, device="cuda").bfloat16()
    slots = (torch.arange(300) + 147_000 * 256 - 300).int().cuda()
    round_trip(cache, k, v, slots)
    assert not cache.read(torch.arange(300, dtype=torch.int32, device="cuda"))[0].any()
    # a request whose tokens lie there
    table = torch.tensor([[146_998, 146_999]], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 2, 256, device="cuda").bfloat16()
    y = cache.attend(q, table, torch.tensor([512], dtype=torch.int32, device="cuda"))
    low = kv.KVCache4(2, 1, 256, page_size=256)
    low.write(k, v, (torch.arange(300) + 212).int().cuda())
    z = low.attend(q, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([512], dtype=torch.int32, device="cuda"))
    assert torch.equal(y, z)
