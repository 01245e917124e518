"""The operators between the projections of a full-attention layer, as measurable cases.

Four operators: rotary positions over several axes (with an optional RMS norm of every head before it),
the step plan of a paged cache (row starts, positions, page assignment, slots, all on the device), the
cache held in 4 bits (rows written and read back), and attention over that cache.

Where `own` is false, run() computes them in elementary torch operations; where it is true, through the
package. Sizes are those of the 9B hybrid model the package is built around (16 query and 4 key/value
heads of 256 elements, 64 of them rotated) or generic ones of the same ranges.

The cache's arithmetic: a row is the D elements of one token and key/value head. lo and hi are its
smallest and largest element, an element's code is rint(15 (x - lo) / (hi - lo)) (half to even), its
value lo + code (hi - lo) / 15.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
THETA = 1e7
EPS = 1e-6
ROWS = 64 * 8192 * 16 * 256               # what the largest decode batch multiplies
SCORES = 16 * 4096 * 8192                 # scores of the largest prompt


def pkg():
    return importlib.import_module("rag-cache-engineering-qwen35-9b-flute_b200")


def listed():
    return [
        # one token of one sequence: rotation with the heads' norms, as every decode step of a single user has it
        dict(name="rotary_one_token", op="rotary", T=1, Hq=16, Hkv=4, D=256, R=64, axes=3, interleaved=True, norm=True,
             gated=True, dtype="bf16", far=131072),
        # a prompt of text and images: three axes, heads normed, queries beside their gates in the projection's rows
        dict(name="rotary_prompt_8192", op="rotary", T=8192, Hq=16, Hkv=4, D=256, R=64, axes=3, interleaved=True,
             norm=True, gated=True, dtype="bf16", far=32768),
        # an odd number of video tokens, whole heads rotated, contiguous sections, no norm
        dict(name="rotary_video_4093", op="rotary", T=4093, Hq=32, Hkv=8, D=128, R=128, axes=3, interleaved=False,
             norm=False, gated=False, dtype="fp16", far=1 << 20),
        # a decode step of eight sequences: eight slots, now and then a new page
        dict(name="plan_decode_8", op="plan", B=8, n=1, cached=8192, page=64),
        # a busy server's step: chunks of prompts among a thousand single tokens
        dict(name="plan_mixed_1024", op="plan", B=1024, n=512, cached=32768, page=16),
        # the keys and values of a decode step of 32 sequences into their pages, and back
        dict(name="cache_decode_32", op="cache", T=32, Hkv=4, D=256, page=64, pages=4096, dtype="bf16"),
        # those of a long prompt
        dict(name="cache_prompt_16384", op="cache", T=16384, Hkv=4, D=256, page=64, pages=4096, dtype="bf16"),
        # one user's token over a long context
        dict(name="attend_1x131072", op="attend", B=1, n=1, L=131072, Hq=16, Hkv=4, D=256, page=64, window=0, sinks=0,
             gate=True, dtype="bf16"),
        # a batch of 64 ragged sequences, one token each
        dict(name="attend_64x8192", op="attend", B=64, n=1, L=8192, Hq=16, Hkv=4, D=256, page=64, window=0, sinks=0,
             gate=True, dtype="bf16"),
        # single tokens over long caches behind a window, the first tokens kept visible
        dict(name="attend_window_16x32768", op="attend", B=16, n=1, L=32768, Hq=32, Hkv=4, D=128, page=32, window=4096,
             sinks=4, gate=False, dtype="fp16"),
        # chunks of prompts of up to 61 rows among single tokens
        dict(name="attend_mixed_16x4096", op="attend", B=16, n=61, L=4096, Hq=24, Hkv=8, D=128, page=16, window=0,
             sinks=0, gate=False, dtype="bf16"),
        # the second half of a long prompt
        dict(name="attend_prompt_4096", op="attend", B=1, n=4096, L=8192, Hq=16, Hkv=4, D=256, page=64, window=0,
             sinks=0, gate=True, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], evenly spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choices(("rotary", "plan", "cache", "attend"), (20, 15, 20, 45))[0]
    dtype = rng.choice(("bf16", "fp16"))
    D = rng.choice((64, 128, 256))
    Hkv = rng.choice((1, 2, 4, 8))
    Hq = Hkv * rng.choice((1, 2, 3, 4, 6, 8))
    page = rng.choice((16, 32, 64, 128))
    if op == "rotary":
        return dict(op=op, T=_log_int(rng, 1, max(1, 8192 * 20 * 256 // ((Hq + Hkv) * D))), Hq=Hq, Hkv=Hkv, D=D,
                    R=rng.choice((D, D // 2, D // 4)), axes=rng.choice((1, 2, 3)), interleaved=rng.random() < 0.5,
                    norm=rng.random() < 0.5, gated=rng.random() < 0.5, dtype=dtype, far=_log_int(rng, 64, 1 << 20))
    if op == "plan":
        return dict(op=op, B=_log_int(rng, 1, 1024), n=_log_int(rng, 1, 512), cached=_log_int(rng, 1, 32768), page=page)
    if op == "cache":
        T = _log_int(rng, 1, min(65536, 16384 * 1024 // (Hkv * D)))
        return dict(op=op, T=T, Hkv=Hkv, D=D, page=page, pages=-(-T // page) + _log_int(rng, 1, 1024), dtype=dtype)
    n = 1 if rng.random() < 0.5 else _log_int(rng, 2, 2048)
    L = max(n, _log_int(rng, 1, 32768))
    B = _log_int(rng, 1, 64)
    B = max(1, min(B, ROWS // (L * max(Hq, 4 * Hkv) * D), SCORES // (Hq * n * L)))
    L = max(1, min(L, SCORES // (Hq * n * B)))
    window = _log_int(rng, 1, L) if rng.random() < 0.3 else 0
    return dict(op="attend", B=B, n=min(n, L), L=L, Hq=Hq, Hkv=Hkv, D=D, page=page, window=window,
                sinks=rng.choice((0, 1, 4, 37)) if window else 0, gate=rng.random() < 0.5, dtype=dtype)


# --------------------------------------------------------------------------- sizes that follow from a case

def _sections(c):
    """Pairs of each axis."""
    half, a = c["R"] // 2, c["axes"]
    return [half - (a - 1) * (half // a)] + [half // a] * (a - 1)


def _lengths(c):
    """Rows and cached tokens with them of each request: ragged, the first one full, the same for every seed."""
    rng = random.Random(c["B"] * 1000003 + c["n"] * 10007 + c["L"])
    rows = [c["n"]] + [_log_int(rng, 1, c["n"]) if c["n"] > 1 else 1 for _ in range(c["B"] - 1)]
    return rows, [c["L"]] + [rng.randint(r, c["L"]) for r in rows[1:]]


def _requests(c):
    """New and cached tokens of each request of a step."""
    rng = random.Random(c["B"] * 1000003 + c["n"] * 10007 + c["cached"])
    new = [_log_int(rng, 1, c["n"]) if rng.random() < 0.25 else 1 for _ in range(c["B"])]
    return new, [rng.randint(0, c["cached"]) for _ in range(c["B"])]


def _visible(length, rows, window, sinks):
    """Cached tokens that some row of a request sees, and (row, token) pairs that are visible."""
    pairs = 0
    for p in range(length - rows, length):
        pairs += p + 1 if not window else min(p + 1, window + min(sinks, max(0, p + 1 - window)))
    if not window:
        return length, pairs
    first = max(0, length - rows - window + 1)
    return length - first + min(sinks, first), pairs


def work(case):
    c = case
    if c["op"] == "rotary":
        moved = 2 * 2 * c["T"] * (c["Hq"] + c["Hkv"]) * c["D"]
        return {"bytes": moved + 8 * c["axes"] * c["T"], "flops": 6.0 * c["T"] * (c["Hq"] + c["Hkv"]) * c["D"]}
    if c["op"] == "plan":
        new, cached = _requests(c)
        pages = sum(-(-(a + b) // c["page"]) - b // c["page"] for a, b in zip(new, cached))
        return {"bytes": 8 * sum(new) + 8 * pages + 17 * c["B"], "flops": 4.0 * (sum(new) + c["B"])}
    if c["op"] == "cache":
        rows = 2 * c["T"] * c["Hkv"]
        return {"bytes": rows * (2 * c["D"] + c["D"] // 2 + 4) + rows * (c["D"] // 2 + 4 + 2 * c["D"]) + 8 * c["T"],
                "flops": 8.0 * rows * c["D"]}
    seen = [_visible(n, r, c["window"], c["sinks"]) for r, n in zip(*_lengths(c))]
    rows = sum(_lengths(c)[0])
    return {"bytes": sum(s for s, _ in seen) * c["Hkv"] * 2 * (c["D"] // 2 + 4)
            + (3 if c["gate"] else 2) * 2 * rows * c["Hq"] * c["D"],
            "flops": 4.0 * c["Hq"] * c["D"] * sum(p for _, p in seen)}


# --------------------------------------------------------------------------- what a program holds before the call

def _randn(g, *shape, dtype):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


def _paged(c, rows, lengths, g):
    """Block table of the requests (pages in no order, unused entries -1) and the number of pages."""
    counts = [-(-n // c["page"]) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    start = torch.tensor(counts, device="cuda").cumsum(0) - torch.tensor(counts, device="cuda")
    at = torch.arange(max(counts), device="cuda")
    inside = at < torch.tensor(counts, device="cuda")[:, None]
    return torch.where(inside, order[(start[:, None] + at).clamp(max=pages - 1)], -1).to(torch.int32).contiguous(), pages


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": c}
    if c["op"] == "rotary":
        dt, T, D = DTYPES[c["dtype"]], c["T"], c["D"]
        wide = 2 * D if c["gated"] else D                     # queries lie beside their gates, head by head
        rows = _randn(g, T, c["Hq"] * wide + c["Hkv"] * D, dtype=dt)
        s["q"] = rows[:, :c["Hq"] * wide].view(T, c["Hq"], wide)[..., :D]
        s["k"] = rows[:, c["Hq"] * wide:].view(T, c["Hkv"], D)
        s["positions"] = torch.randint(0, c["far"], (c["axes"], T), device="cuda", generator=g)
        if c["norm"]:
            s["q_gain"] = (1 + 0.1 * _randn(g, D, dtype=torch.float32)).to(dt)
            s["k_gain"] = (1 + 0.1 * _randn(g, D, dtype=torch.float32)).to(dt)
        if own:
            s["rotary"] = pkg().rotary.AxisRotary(c["R"], theta=THETA, sections=_sections(c),
                                                  interleaved=c["interleaved"])
        return s
    if c["op"] == "plan":
        new, cached = _requests(c)
        page = c["page"]
        s["new"], s["cached"] = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (new, cached))
        have = [-(-n // page) for n in cached]
        want = [-(-(a + b) // page) for a, b in zip(new, cached)]
        width, pages = max(want) + 2, sum(want) + 64
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        first = torch.tensor(have, device="cuda").cumsum(0) - torch.tensor(have, device="cuda")
        at = torch.arange(width, device="cuda")
        inside = at < torch.tensor(have, device="cuda")[:, None]
        s["block_table"] = torch.where(inside, order[(first[:, None] + at).clamp(max=pages - 1)], -1).to(torch.int32)
        s["free_pages"] = order[sum(have):].contiguous()
        s["taken"] = torch.randint(0, 32, (1,), device="cuda", generator=g).to(torch.int32)
        s["max_tokens"] = -(-sum(new) // 256) * 256           # the step's buffers are padded
        return s
    dt, D, H, page = DTYPES[c["dtype"]], c["D"], c["Hkv"], c["page"]
    if c["op"] == "cache":
        s["k"] = (_randn(g, c["T"], H, D, dtype=torch.float32) + _randn(g, H, D, dtype=torch.float32)).to(dt)
        s["v"] = _randn(g, c["T"], H, D, dtype=dt)
        s["slots"] = torch.randperm(c["pages"] * page, device="cuda", generator=g)[:c["T"]].to(torch.int32)
        if c["T"] > 64:                                       # a prompt fills its pages in order
            start = torch.randperm(c["pages"], device="cuda", generator=g)[:-(-c["T"] // page), None] * page
            s["slots"] = (start + torch.arange(page, device="cuda")).reshape(-1)[:c["T"]].to(torch.int32)
        if own:
            s["cache"] = pkg().kvcache.KVCache4(c["pages"], H, D, page_size=page, dtype=dt)
        else:
            s["codes"] = torch.zeros(2, c["pages"] * page, H, D, dtype=torch.uint8, device="cuda")
            s["range"] = torch.zeros(2, c["pages"] * page, H, 2, dtype=dt, device="cuda")
        return s
    rows, lengths = _lengths(c)
    s["block_table"], pages = _paged(c, rows, lengths, g)
    s["kv_len"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    s["row_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    s["q"] = 2 * _randn(g, start[-1], c["Hq"], D, dtype=dt)
    if c["gate"]:
        s["gate"] = _randn(g, start[-1], c["Hq"], D, dtype=dt)
    k = _randn(g, pages * page, H, D, dtype=dt) + _randn(g, H, D, dtype=dt)
    v = _randn(g, pages * page, H, D, dtype=dt)
    if own:
        s["cache"] = pkg().kvcache.KVCache4(pages, H, D, page_size=page, dtype=dt)
        s["cache"].write(k, v, torch.arange(pages * page, dtype=torch.int32, device="cuda"))
    else:
        s["codes"], s["range"] = (torch.stack(x) for x in zip(_codes(k), _codes(v)))
    return s


# --------------------------------------------------------------------------- the plain forms

def _codes(x):
    """Codes (uint8) and the pair (lo, hi) of every row."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    a = 15.0 * (x.float() - lo.float())
    b = hi.float() - lo.float()
    return torch.where(b > 0, torch.round(a / b), torch.zeros_like(a)).to(torch.uint8), torch.cat((lo, hi), -1)


def _values(codes, pair):
    """fp32 values of codes under their pair (lo, hi)."""
    lo, hi = pair[..., :1].float(), pair[..., 1:].float()
    return lo + codes.float() * ((hi - lo) / 15.0)


def _axis_of_pair(c):
    half, sec = c["R"] // 2, _sections(c)
    if not c["interleaved"]:
        return torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(sec))
    i = torch.arange(half)
    a = i % c["axes"]
    return torch.where(i < c["axes"] * torch.tensor(sec)[a], a, torch.zeros_like(a))


def _rotate(x, cos, sin, gain, R):
    x = x.float()
    if gain is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain.float()
    a, b = x[..., :R // 2], x[..., R // 2:R]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., R:]), -1)


def _plain_rotary(s):
    c = s["case"]
    R = c["R"]
    freq = THETA ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    angle = s["positions"].double()[_axis_of_pair(c).cuda()].T * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    dt = DTYPES[c["dtype"]]
    return [_rotate(s[n], cos, sin, s.get(n + "_gain"), R).to(dt) for n in ("q", "k")]


def _plain_plan(s):
    page, width, room = s["case"]["page"], s["block_table"].shape[1], s["max_tokens"]
    new, cached = s["new"].long().clamp(min=0), s["cached"].long().clamp(min=0)
    end = new.cumsum(0)
    start = (end - new).clamp(max=room)
    have, want = (cached + page - 1) // page, (cached + new + page - 1) // page
    fits = (want <= width) & (end <= room)
    need = torch.where(fits, want - have, torch.zeros_like(want))
    upto = s["taken"].long() + need.cumsum(0)
    served = fits & ((need == 0) | (upto <= s["free_pages"].numel()))
    taken = torch.maximum(s["taken"].long(), torch.where(served & (need > 0), upto, torch.zeros_like(upto)).amax())
    at = torch.arange(width, device="cuda")
    fresh = served[:, None] & (at >= have[:, None]) & (at < want[:, None])
    index = (upto - need - have)[:, None] + at
    table = torch.where(fresh, s["free_pages"][index.clamp(0, s["free_pages"].numel() - 1)], s["block_table"])
    t = torch.arange(room, device="cuda")
    b = torch.searchsorted(end, t, right=True).clamp(max=new.numel() - 1)
    live = t < end[-1]
    pos = torch.where(live, cached[b] + t - (end - new)[b], torch.zeros_like(t))
    entry = table[b, (pos // page).clamp(max=width - 1)]
    slots = torch.where(live & served[b] & (entry >= 0), entry.long() * page + pos % page, -torch.ones_like(t))
    s["block_table"].copy_(table)
    row_start = torch.cat((start, end[-1:].clamp(max=room)))
    return {"row_start": row_start.int(), "kv_len": torch.where(served, cached + new, cached).int(),
            "positions": pos.int(), "slots": slots.int(), "taken": taken.int(), "served": served,
            "block_table": s["block_table"]}


def _plain_cache(s):
    at = s["slots"].long()
    out = []
    for i, x in enumerate((s["k"], s["v"])):
        s["codes"][i][at], s["range"][i][at] = _codes(x)
        out.append(_values(s["codes"][i][at], s["range"][i][at]).to(x.dtype))
    return out


def _plain_attend(s):
    c = s["case"]
    B, Hq, H, D, page = c["B"], c["Hq"], c["Hkv"], c["D"], c["page"]
    G, n, L = Hq // H, c["n"], c["L"]
    table = s["block_table"].long().clamp(min=0)
    token = (table[:, :, None] * page + torch.arange(page, device="cuda")).reshape(B, -1)[:, :L]       # [B, L]
    rows = s["row_start"].long()
    i = torch.arange(n, device="cuda")
    inside = i < (rows[1:] - rows[:-1])[:, None]                                                        # [B, n]
    at = (rows[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].float().view(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    k = _values(s["codes"][0][token], s["range"][0][token]).transpose(1, 2)                             # [B, H, L, D]
    p = torch.matmul(q, k.transpose(2, 3)).mul_(1 / math.sqrt(D)).view(B, H, G, n, L)
    del k
    j = torch.arange(L, device="cuda")
    pos = s["kv_len"].long()[:, None] - (rows[1:] - rows[:-1])[:, None] + i                             # [B, n]
    seen = (j <= pos[..., None]) & inside[..., None]
    if c["window"]:
        seen &= (j > pos[..., None] - c["window"]) | (j < c["sinks"])
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = _values(s["codes"][1][token], s["range"][1][token]).transpose(1, 2)
    o = torch.matmul(p.view(B, H, G * n, L), v).view(B, H, G, n, D)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    t = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(rows[1:], t, right=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)[b, t - rows[b]]
    if c["gate"]:
        o = o / (1 + torch.exp(-s["gate"].float()))
    return o.to(DTYPES[c["dtype"]])


# --------------------------------------------------------------------------- one pass

def _own_rotary(s):
    return list(s["rotary"](s["q"], s["k"], s["positions"], q_gain=s.get("q_gain"), k_gain=s.get("k_gain"), eps=EPS))


def _own_plan(s):
    p = pkg().kvcache.plan_step(s["cached"], s["new"], s["block_table"], s["free_pages"], s["taken"],
                                page_size=s["case"]["page"], max_tokens=s["max_tokens"])
    return {"row_start": p.row_start, "kv_len": p.kv_len, "positions": p.positions, "slots": p.slots, "taken": p.taken,
            "served": p.served, "block_table": s["block_table"]}


def _own_cache(s):
    s["cache"].write(s["k"], s["v"], s["slots"])
    return list(s["cache"].read(s["slots"]))


def _own_attend(s):
    c = s["case"]
    # one row per request needs no row starts
    return s["cache"].attend(s["q"], s["block_table"], s["kv_len"], row_start=None if c["n"] == 1 else s["row_start"],
                             window=c["window"], sinks=c["sinks"], gate=s.get("gate"))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "plan": _own_plan, "cache": _own_cache, "attend": _own_attend}[op](state)
    return {"rotary": _plain_rotary, "plan": _plain_plan, "cache": _plain_cache, "attend": _plain_attend}[op](state)


# --------------------------------------------------------------------------- 64 bits, from the definitions

def _row_values64(x):
    """What the 4-bit cache makes of rows x."""
    x = x.double()
    lo = x.amin(-1, keepdim=True)
    width = x.amax(-1, keepdim=True) - lo
    q = torch.where(width > 0, torch.round(15 * (x - lo) / width), torch.zeros_like(x))
    return lo + q * width / 15


def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None                                     # whole numbers: held to equality
    if c["op"] == "attend":
        s = _attend_inputs(c, seed)
        rows, lengths = _lengths(c)
        G, out, r0 = c["Hq"] // c["Hkv"], [], 0
        for b, (n, length) in enumerate(zip(rows, lengths)):
            pages = s["block_table"][b, :-(-length // c["page"])].long()
            tok = (pages[:, None] * c["page"] + torch.arange(c["page"], device="cuda")).flatten()[:length]
            k, v = _row_values64(s["k"][tok]), _row_values64(s["v"][tok])
            q = s["q"][r0:r0 + n].double()
            pos = torch.arange(length - n, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")[None]
            hidden = j > pos
            if c["window"]:
                hidden = hidden | ((pos - j >= c["window"]) & (j >= c["sinks"]))
            heads = []
            for h in range(c["Hq"]):
                logits = (q[:, h] @ k[:, h // G].T) / c["D"] ** 0.5
                logits[hidden] = -math.inf
                heads.append(torch.softmax(logits, -1) @ v[:, h // G])
            out.append(torch.stack(heads, 1))
            r0 += n
        out = torch.cat(out)
        return out * torch.sigmoid(s["gate"].double()) if c["gate"] else out
    s = prepare(c, seed)
    if c["op"] == "cache":
        return [_row_values64(s["k"]), _row_values64(s["v"])]
    R, sec, out = c["R"], _sections(c), []
    axis = []
    if c["interleaved"]:
        for i in range(R // 2):
            a = i % c["axes"]
            axis.append(a if i < c["axes"] * sec[a] else 0)
    else:
        for a, count in enumerate(sec):
            axis += [a] * count
    for name in ("q", "k"):
        x = s[name].double()
        if c["norm"]:
            x = x / (x.square().sum(-1, keepdim=True) / c["D"] + EPS).sqrt() * s[name + "_gain"].double()
        y = x.clone()
        for i in range(R // 2):
            turn = s["positions"][axis[i]].double() / THETA ** (2 * i / R)
            z = torch.polar(torch.ones_like(turn), turn)[:, None] * torch.complex(x[..., i], x[..., i + R // 2])
            y[..., i], y[..., i + R // 2] = z.real, z.imag
        out.append(y)
    return out


def _attend_inputs(c, seed):
    """The inputs of prepare(c, seed) with the keys and values as they were before they were coded."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]
    rows, lengths = _lengths(c)
    s = {}
    s["block_table"], pages = _paged(c, rows, lengths, g)
    s["q"] = 2 * _randn(g, sum(rows), c["Hq"], c["D"], dtype=dt)
    if c["gate"]:
        s["gate"] = _randn(g, sum(rows), c["Hq"], c["D"], dtype=dt)
    s["k"] = _randn(g, pages * c["page"], c["Hkv"], c["D"], dtype=dt) + _randn(g, c["Hkv"], c["D"], dtype=dt)
    s["v"] = _randn(g, pages * c["page"], c["Hkv"], c["D"], dtype=dt)
    return s
