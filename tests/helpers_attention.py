"""64-bit restatements of the attention side (rotary positions, the 4-bit cache, attention over it) for the
GPU tests, and how far a result may lie from them.

Rounding to a 16-bit type is off by at most half a step, u = eps / 2 relative to the value (bf16 2^-8, fp16
2^-11), and by half the smallest subnormal below the normal range.
"""
from __future__ import annotations

import math

import torch


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def floor(dtype):
    """Half the smallest subnormal."""
    info = torch.finfo(dtype)
    return info.smallest_normal * info.eps / 2


def values64(x):
    """What a 4-bit row makes of x [..., D]: lo + rint(15 (x - lo) / (hi - lo)) (hi - lo) / 15."""
    x = x.double()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    code = torch.where(hi > lo, torch.round(15 * (x - lo) / (hi - lo)), torch.zeros_like(x))
    v = lo + code * (hi - lo) / 15
    return torch.where((hi - lo).isfinite() & ((hi - lo) < 2.0 ** 120), v, torch.full_like(v, math.nan))


def visible(pos, length, window, sinks):
    """[rows, length] truth values for rows at positions pos."""
    j = torch.arange(length, device=pos.device)
    see = j <= pos[:, None]
    if window:
        see = see & ((j > pos[:, None] - window) | (j < sinks))
    return see


def attend64(q, k, v, pos, scale, window=0, sinks=0, gate=None):
    """q [rows, Hq, D], k and v [length, H, D] (the values that the cache stands for, or NaN), pos [rows].
    Returns the result in 64 bits and the bound of its error."""
    rows, Hq, D = q.shape
    L, H, _ = k.shape
    out = torch.zeros(rows, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    see = visible(pos, L, window, sinks)
    u = unit(q.dtype)
    for h in range(Hq):
        kk, vv, qq = k[:, h // (Hq // H)].double(), v[:, h // (Hq // H)].double(), q[:, h].double()
        kk, vv = torch.where(see.any(0)[:, None], kk, 0.0), torch.where(see.any(0)[:, None], vv, 0.0)
        if L:
            s = (qq @ kk.T) * scale
            s = torch.where(see, s, -math.inf)
            some = see.any(1, keepdim=True)
            p = torch.where(some, torch.softmax(s, -1), torch.zeros_like(s))
            o = p @ torch.where(see.any(0)[:, None], vv, 0.0)
            # The scores: at most 16 fp32 sums of products q c in a row, each off by 2^-23 of at most
            # |q|_1 range, and lo sum(q): together below 2^-20 scale |q|_1 (|lo| + range); a probability moves by
            # twice that. p * step is rounded to fp16: 2^-12 of a sum that is at most the values' range,
            # and 2^-25 a token where it is subnormal. The sum over tokens adds 2^-26 a token (one in 16 rounds).
            def spread(x):
                return (x.amax(-1) - x.amin(-1)).nan_to_num().amax().item(), x.abs().nan_to_num().amax().item()
            kr, km = spread(kk)
            vr, vm = spread(vv)
            reach = 2.0 ** -19 * abs(scale) * qq.abs().sum(-1, keepdim=True) * (kr + km)
            err = (vr + 2.0 ** -10 * vm) * (2.0 ** -12 + L * 2.0 ** -24 + reach)
        else:
            o, err = torch.zeros_like(qq), torch.zeros_like(qq[:, :1])
        if gate is not None:
            o = o * torch.sigmoid(gate[:, h].double())
        out[:, h] = o
        tol[:, h] = err + (u + 2.0 ** -20) * o.abs() + floor(q.dtype)
    return out, tol


def rotate64(x, positions, R, theta, axis_of_pair, gain=None, eps=1e-6):
    """x [T, heads, D] rotated, and the bound of its error: cos and sin are off by 2^-22 (a 32-bit turn and a
    32-bit sine), the products and the norm by 2^-22 of the two elements of a pair."""
    y = x.double()
    if gain is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * gain.double()
    freq = theta ** (-torch.arange(0, R, 2, dtype=torch.float64, device=x.device) / R)
    ang = positions.double()[axis_of_pair.to(x.device).long()].T * freq
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = y[..., :R // 2], y[..., R // 2:R]
    out = torch.cat((a * c - b * s, b * c + a * s, y[..., R:]), -1)
    size = torch.cat((a.abs() + b.abs(), a.abs() + b.abs(), y[..., R:].abs()), -1)
    return out, unit(x.dtype) * out.abs() + 2.0 ** -20 * size + floor(x.dtype)


def close(got, want, tol, what=""):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in {int((got.isnan() != want.isnan()).sum())} other places"
    off = ((got - want).abs() / tol).nan_to_num(0.0)
    assert off.numel() == 0 or off.max().item() <= 1, f"{what}: off by {off.max().item():.3g} times the bound"
