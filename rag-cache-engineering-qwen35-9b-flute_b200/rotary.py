"""Rotary positions over several axes (time, height, width), served by the CUDA library.

Elements (i, i + R/2), i < R/2, of each head turn by positions[axis(i), t] * theta^(-2i/R); the other
elements of a head pass. With gains, each head is first normed: x * rsqrt(mean(x^2) + eps) * gain.
fp32 inside (the angle's whole turns are dropped in fp64), one rounding.
"""
from __future__ import annotations

import ctypes
import math
import threading
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ["AxisRotary"]


def rows16(x: torch.Tensor) -> torch.Tensor:
    """x [T, heads, D] as the kernels read it: 16-byte rows, any token and head stride (a copy where
    its strides or its address do not allow that)."""
    if x.shape[0] == 1 or x.shape[1] == 1:          # the stride of a single token or head says nothing, and may be anything
        token, head = (0 if n == 1 else s for n, s in zip(x.shape[:2], x.stride()))
        if (token, head) != x.stride()[:2]:
            x = x.as_strided(x.shape, (token, head, x.stride(2)))
    if x.stride(2) == 1 and x.stride(0) % 8 == 0 and x.stride(1) % 8 == 0 and x.data_ptr() % 16 == 0:
        return x
    return torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)


def check_no_grad(name: str, x: torch.Tensor) -> None:
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires grad: autograd is not served on the attention side")
    if torch._C._is_fwd_grad_enabled() and forward_ad.unpack_dual(x).tangent is not None:
        raise RuntimeError(f"{name} carries a forward-mode tangent: autograd is not served on the attention side")


def check_heads(name: str, x: torch.Tensor, heads: Optional[int], D: Optional[int]) -> None:
    _lib._need_cuda(x, name)
    if x.dim() != 3 or (heads is not None and x.shape[1] != heads) or (D is not None and x.shape[2] != D):
        raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, "
                         f"{'head_dim' if D is None else D}], got {tuple(x.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name} must be bfloat16 or float16, got {x.dtype}")
    check_no_grad(name, x)


class AxisRotary:
    """The rotation of one model: rotary_dim R (a multiple of 16 up to head_dim), theta, and how many of
    the R/2 pairs turn with each axis. sections=(a, b, c) gives the first a pairs to axis 0, the next b to
    axis 1 and so on; interleaved deals them in turn: pair i turns with axis x = i % axes while
    i < axes * sections[x], the rest with axis 0. Without sections there is one axis.

        rot = AxisRotary(64, theta=1e7, sections=(12, 10, 10), interleaved=True)
        q, k = rot(q, k, positions)            # positions [3, tokens], or [tokens] for all axes
    """

    def __init__(self, rotary_dim: int, theta: float = 10000.0, sections: Optional[Sequence[int]] = None,
                 interleaved: bool = False):
        R = int(rotary_dim)
        if R < 16 or R % 16 or R > 256:
            raise ValueError(f"rotary_dim must be a multiple of 16 from 16 to 256, got {rotary_dim}")
        if not (theta > 0 and math.isfinite(theta)):
            raise ValueError(f"theta must be positive, got {theta}")
        sections = [R // 2] if sections is None else [int(s) for s in sections]
        if not sections or min(sections) < 0 or sum(sections) != R // 2:
            raise ValueError(f"sections must add up to rotary_dim / 2 = {R // 2}, got {sections}")
        n = len(sections)
        if interleaved:
            axis = [i % n if i < n * sections[i % n] else 0 for i in range(R // 2)]
            if any(axis.count(a) != s for a, s in enumerate(sections)):
                raise ValueError(f"sections {sections} cannot be interleaved over {R // 2} pairs")
        else:
            axis = [a for a, s in enumerate(sections) for _ in range(s)]
        self.rotary_dim, self.theta, self.sections, self.interleaved = R, float(theta), tuple(sections), bool(interleaved)
        self.axes = n
        self.axis = torch.tensor(axis, dtype=torch.int32)
        self.turns = (theta ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)) / (2 * math.pi)
        self._tables, self._lock = {}, threading.Lock()

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_tables", "_lock")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._tables, self._lock = {}, threading.Lock()

    def _on(self, device: torch.device):
        """Turns and axes on `device` (copied once, before any capture needs them)."""
        t = self._tables.get(device)
        if t is None:
            with self._lock:
                t = (self.turns.to(device), self.axis.to(device))
                torch.cuda.current_stream(device).synchronize()      # other streams use them too
                self._tables[device] = t
        return t

    def to(self, device) -> "AxisRotary":
        """Puts the tables on `device` now (a first call inside a stream capture could not)."""
        device = torch.device(device)
        self._on(torch.device("cuda", torch.cuda.current_device()) if device.type == "cuda" and device.index is None
                 else device)
        return self

    def __call__(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, q_gain: Optional[torch.Tensor] = None,
                 k_gain: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
        """q [tokens, heads, D] and k [tokens, kv_heads, D], D in {64, 128, 256}, rotated into new
        contiguous tensors. positions: int32 or int64, [axes, tokens] or [tokens]. q_gain, k_gain: [D] in
        q's dtype, both or neither. Nothing is differentiated: inputs and gains that require grad are refused
        while grad mode is on."""
        tables = self._tables.get(q.device)
        if tables is not None:
            done = _lib.host.rotary(q, k, positions, q_gain, k_gain, eps, *tables, self.axes)
            if done is not None:
                return done
        check_heads("q", q, None, None)
        check_heads("k", k, None, q.shape[2])
        T, Hq, D = q.shape
        if k.shape[0] != T or k.dtype != q.dtype or k.device != q.device:
            raise ValueError("k must have q's tokens, dtype and device")
        if positions.device != q.device or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("positions must be an int32 or int64 tensor on q's device")
        if tuple(positions.shape) not in ((T,), (self.axes, T)):
            raise ValueError(f"positions must be [{T}] or [{self.axes}, {T}], got {tuple(positions.shape)}")
        if (q_gain is None) != (k_gain is None):
            raise ValueError("q_gain and k_gain come together")
        if q_gain is not None:
            for name, g in (("q_gain", q_gain), ("k_gain", k_gain)):
                if tuple(g.shape) != (D,) or g.dtype != q.dtype or g.device != q.device:
                    raise ValueError(f"{name} must be [{D}] in q's dtype on q's device")
                check_no_grad(name, g)
            q_gain, k_gain = (g.contiguous() if g.data_ptr() % 16 == 0 else g.clone() for g in (q_gain, k_gain))
        q, k = rows16(q), rows16(k)
        if positions.stride(-1) != 1 and T > 1:
            positions = positions.contiguous()
        turns, axis = self._on(q.device)
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=q.dtype, device=q.device)
        a = _lib.RotaryArgs(
            q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), _lib.ptr(q_gain), _lib.ptr(k_gain),
            positions.data_ptr(), turns.data_ptr(), axis.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1),
            positions.stride(0) if positions.dim() == 2 else 0, T, Hq, k.shape[1], D, self.rotary_dim,
            int(positions.dtype == torch.int64), _lib.dtype_id(q.dtype), float(eps))
        if T:
            with _lib._on_device(q.device):
                _lib.check(_lib.lib().b200lut_rotary(ctypes.byref(a), _lib._stream(q)))
        return q_out, k_out
