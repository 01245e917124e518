"""A full-attention layer over the 4-bit cache: merged Q/K/V projection, rotary positions (with an optional norm of
every head), cache rows, attention, output projection.

    attn = PalettizedAttention(SplitQKV(q, k, v), o, AxisRotary(64, theta=1e7), head_dim=256, gated=True)
    step = plan_step(kv_len, fresh, block_table, free_pages, taken, cache.page_size, max_tokens=x.shape[0])
    y = attn(x, cache, block_table, step)                       # prompts, chunks and single tokens mixed
    y = attn(x, cache, block_table, step, one_row_each=True)    # decode: row b is request b's one token

One step plan serves every layer of a model; each layer has a cache of its own. No call waits for the GPU, and a
step can be captured into a CUDA graph (the rotation's tables are on the device after the first call, or
AxisRotary.to).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from .kvcache import KVCache4, StepPlan
from .rotary import AxisRotary

__all__ = ["PalettizedAttention", "attend_projected"]


def attend_projected(qkv: torch.Tensor, n_heads: int, cache: KVCache4, block_table: torch.Tensor, step: StepPlan,
                     rotary: AxisRotary, positions: Optional[torch.Tensor] = None, gated: bool = False,
                     q_gain: Optional[torch.Tensor] = None, k_gain: Optional[torch.Tensor] = None, eps: float = 1e-6,
                     scale: Optional[float] = None, window: int = 0, sinks: int = 0, one_row_each: bool = False,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What lies between the projections: qkv [tokens, q | k | v] -> [tokens, n_heads, head_dim]. q holds head_dim
    elements a head, or, gated, head_dim of the query and then head_dim of the gate. The parts are read where they
    lie, without copies."""
    D, H = cache.head_dim, cache.n_kv_heads
    nq, nk = n_heads * D * (2 if gated else 1), H * D
    if qkv.dim() != 2 or qkv.shape[1] != nq + 2 * nk:
        raise ValueError(f"qkv must be [tokens, {nq} + 2 * {nk}], got {tuple(qkv.shape)}")
    T = qkv.shape[0]
    if step.slots.shape[0] != T:
        raise ValueError(f"the step plan is for {step.slots.shape[0]} rows, got {T}")
    if one_row_each and step.kv_len.shape[0] != T:
        raise ValueError(f"one_row_each: {T} rows, {step.kv_len.shape[0]} requests")
    q = qkv[:, :nq].unflatten(1, (n_heads, nq // n_heads))
    k, v = (qkv[:, nq + i * nk:nq + (i + 1) * nk].unflatten(1, (H, D)) for i in range(2))
    qr, kr = rotary(q[..., :D], k, step.positions if positions is None else positions, q_gain, k_gain, eps)
    cache.write(kr, v, step.slots)
    return cache.attend(qr, block_table, step.kv_len, None if one_row_each else step.row_start, scale=scale, window=window,
                        sinks=sinks, gate=q[..., D:] if gated else None, out=out)


class PalettizedAttention(nn.Module):
    """o_proj(attention(rotary(q), rotary(k), v)) of x [tokens, K] with the requests' earlier tokens in a cache.

    qkv: a SplitQKV whose q_proj gives n_heads * head_dim rows, or, gated, 2 * head_dim a head: the query and then a
    gate by whose sigmoid the head's result is multiplied. q_gain, k_gain [head_dim]: gains of an RMS norm of every
    head in front of the rotation (both or neither; detached, or under no_grad: nothing is differentiated). window, sinks,
    scale: as KVCache4.attend."""

    def __init__(self, qkv, o_proj, rotary: AxisRotary, head_dim: int, gated: bool = False,
                 q_gain: Optional[torch.Tensor] = None, k_gain: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 scale: Optional[float] = None, window: int = 0, sinks: int = 0):
        super().__init__()
        D, per = int(head_dim), int(head_dim) * (2 if gated else 1)
        if D not in (64, 128, 256):
            raise ValueError(f"PalettizedAttention: head_dim must be 64, 128 or 256, got {head_dim}")
        nq, nk, nv = qkv.q_proj.N, qkv.k_proj.N, qkv.v_proj.N
        if nq % per or nk % D or nk != nv or (nq // per) % (nk // D) or nq // per > 64 * (nk // D):
            raise ValueError(f"PalettizedAttention: q, k and v projections of {nq}, {nk} and {nv} rows do not make up to 64 query "
                             f"heads of {per} for each key and value head of {D}")
        self.n_heads, self.n_kv_heads, self.head_dim = nq // per, nk // D, D
        if o_proj.K != self.n_heads * D:
            raise ValueError(f"PalettizedAttention: o_proj reads {o_proj.K} columns, {self.n_heads} heads of {D} give "
                             f"{self.n_heads * D}")
        if rotary.rotary_dim > D:
            raise ValueError(f"PalettizedAttention: rotary_dim {rotary.rotary_dim} is larger than head_dim {D}")
        if (q_gain is None) != (k_gain is None):
            raise ValueError("PalettizedAttention: q_gain and k_gain come together")
        for name, g in (("q_gain", q_gain), ("k_gain", k_gain)):
            if g is not None and tuple(g.shape) != (D,):
                raise ValueError(f"PalettizedAttention: {name} must be [{D}], got {tuple(g.shape)}")
            self.register_buffer(name, g, persistent=False)
        if window < 0 or sinks < 0:
            raise ValueError("PalettizedAttention: window and sinks must not be negative")
        self.qkv, self.o_proj, self.rotary = qkv, o_proj, rotary
        self.gated, self.eps, self.scale, self.window, self.sinks = bool(gated), float(eps), scale, int(window), int(sinks)

    def forward(self, x: torch.Tensor, cache: KVCache4, block_table: torch.Tensor, step: StepPlan,
                positions: Optional[torch.Tensor] = None, one_row_each: bool = False) -> torch.Tensor:
        """x [tokens, K] -> [tokens, o_proj.N], row t at step.positions[t] (or positions [axes, tokens]); the rows' keys
        and values are written to the cache first. Rows behind the plan's last one come out as o_proj of zeros, whatever
        x holds there; those of a request that was not served mean nothing. With one_row_each every request has exactly
        one row (step.row_start is then not read)."""
        if x.dim() != 2:
            raise ValueError(f"PalettizedAttention: x must be [tokens, {self.qkv.q_proj.K}], got {tuple(x.shape)}")
        if cache.n_kv_heads != self.n_kv_heads or cache.head_dim != self.head_dim or cache.dtype != x.dtype:
            raise ValueError(f"PalettizedAttention: the cache holds {cache.n_kv_heads} heads of {cache.head_dim} in {cache.dtype}, "
                             f"the layer makes {self.n_kv_heads} of {self.head_dim} in {x.dtype}")
        out = None if one_row_each else torch.zeros(x.shape[0], self.n_heads, self.head_dim, dtype=x.dtype, device=x.device)
        y = attend_projected(self.qkv(x), self.n_heads, cache, block_table, step, self.rotary, positions, self.gated,
                             self.q_gain, self.k_gain, self.eps, self.scale, self.window, self.sinks, one_row_each, out)
        return self.o_proj(y.flatten(1))
