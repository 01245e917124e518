"""How far attention over the 4-bit cache may lie from its definition, from a row's own weights (helpers_attention.attend64
bounds it by the largest range of values in the sequence times its length, which a long sequence's lost part can hide in).

For one row with weights p_j over the tokens it sees, values of range r_j (fifteen steps) around a middle, S = sum p_j r_j:
  - w_j = p_j step_j is rounded to fp16, 2^-11 of it, and acts on a code less 7.5 or 8, at most 8/15 of r_j: 2^-11 (8/15) S;
    weights 2^-29 below the row's largest are subnormal: another 2^-30 of the largest p_j r_j a token.
  - a product that the tensor core adds keeps 2^-15 of the largest factor of its group of 16 tokens (codes are subnormal
    halves, whose alignment counts ten bits they do not have): 16 2^-15 w a group, 2^-11 / 15 S.
  - fp32 sums: one in 16 tokens rounds, 2^-24 of at most S: L 2^-28 S; 2^-20 (|lo| + r_j) for middles, join and division.
  - scores: 2^-20 scale |q|_1 (|lo| + range) for sums and parameters, 2^-23 of the score for its difference from the
    maximum, and the same alignment, 2^-15 max|q| step an element; a weight moves by twice that, times |v_j - o|.
"""
from __future__ import annotations

import torch

from helpers_attention import floor, unit, visible


def attend_tight(q, k, v, pos, scale, window=0, sinks=0, split=False):
    """As helpers_attention.attend64. split: weights are held in two halves (2^-22 instead of 2^-11)."""
    rows, Hq, D = q.shape
    L, H, _ = k.shape
    out = torch.zeros(rows, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    see = visible(pos, L, window, sinks)
    for h in range(Hq):
        kk, vv, qq = k[:, h // (Hq // H)].double(), v[:, h // (Hq // H)].double(), q[:, h].double()
        s = torch.where(see, (qq @ kk.T) * scale, -torch.inf)
        p = torch.where(see.any(1, keepdim=True), torch.softmax(s, -1), 0.0)
        o = p @ vv
        r = vv.amax(-1) - vv.amin(-1)
        kr = torch.where(see.any(0), kk.amax(-1) - kk.amin(-1), 0.0).amax()
        km = torch.where(see.any(0)[:, None], kk, 0.0).abs().amax()
        S = p @ r
        reach = abs(scale) * (2.0 ** -20 * qq.abs().sum(-1) * (kr + km) + 2.0 ** -15 * D * qq.abs().amax(-1) * kr / 15)
        reach = reach + 2.0 ** -23 * torch.where(see, s, 0.0).abs().amax(-1)
        spread = p @ vv.abs() + o.abs() * p.sum(-1, keepdim=True)
        err = S * ((2.0 ** -22 if split else 2.0 ** -11) * 8 / 15 + 2.0 ** -11 / 15 + L * 2.0 ** -28)
        err = err + L * 2.0 ** -30 * (p * r).amax(-1) + 2.0 ** -20 * (p @ (vv.abs().amax(-1) + r))
        out[:, h] = o
        tol[:, h] = err[:, None] + 2 * reach[:, None] * spread + (unit(q.dtype) + 2.0 ** -20) * o.abs() + floor(q.dtype)
    return out, tol


def counted_values(L, D):
    """Values [L, D] by which a result counts its tokens: all of 16-token tile t is 8 at element t % D, -7 at t + 1 and 0
    elsewhere (fifteen steps of 1). Under equal weights a tile's absence moves an element by 128 / L."""
    v = torch.zeros(L, D, dtype=torch.float64)
    t = torch.arange(L) // 16
    v[torch.arange(L), t % D], v[torch.arange(L), (t + 1) % D] = 8, -7
    return v


def counted_want(v, lengths, dtype):
    """Means of the first lengths[i] of counted_values, and their bound. All weights of a row are alike, so their rounding
    to fp16 is one factor, 2^-11, of what codes are away from 7.5 or 8 on average, which is at most 1 plus the mean; fp32
    sums of parts: 2^-18 of that; 2^-20 of the parameters' sizes; the result's rounding."""
    total = v.cumsum(0)[lengths - 1]
    want = total / lengths[:, None]
    tol = (2.0 ** -11 + 2.0 ** -18) * (1 + want.abs()) + 2.0 ** -20 * 8 + unit(dtype) * want.abs() + floor(dtype)
    return want, tol
