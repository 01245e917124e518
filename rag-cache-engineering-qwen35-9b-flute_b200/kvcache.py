"""A paged key/value cache held in 4 bits, the step plan that feeds it, and attention over it.

    cache = KVCache4(n_pages, n_kv_heads, head_dim, page_size=64)
    step = plan_step(cached, fresh, block_table, free_pages, taken, page_size=64, max_tokens=T)
    cache.write(k, v, step.slots)
    y = cache.attend(q, block_table, step.kv_len, step.row_start)

A row is the head_dim elements of one token and key/value head: its smallest and largest element lo and hi are
kept exactly, an element is the code rint(15 (x - lo) / (hi - lo)) (half to even) and stands for lo + code (hi -
lo) / 15. A row with a NaN, an infinity or a range of 2^120 and more reads as NaN. Rows whose elements are
spread evenly lose least: rotate heads with outlier elements first (fht.fht_block on queries and keys alike
leaves every score as it is).

Everything that follows the requests' lengths is on the device: no call waits for the GPU, and all of them
can be captured into CUDA graphs.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .rotary import check_heads, check_no_grad, rows16

__all__ = ["KVCache4", "StepPlan", "plan_step"]

PAGE_SIZES = (16, 32, 64, 128, 256)
INT_MAX = 2 ** 31 - 1


class StepPlan(NamedTuple):
    """What a step needs: row_start [B + 1] (rows of request b: row_start[b] .. row_start[b + 1]), kv_len [B]
    (tokens of the request with the new ones), positions and slots [max_tokens] (0 and -1 behind the last
    row), taken [1] (entries of the free list used so far), served [B] (bool)."""
    row_start: torch.Tensor
    kv_len: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    taken: torch.Tensor
    served: torch.Tensor


def _ints(name: str, t: torch.Tensor, shape, device) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != device or t.dim() != len(shape) or \
            any(w is not None and w != n for w, n in zip(shape, t.shape)):
        want = ", ".join("*" if w is None else str(w) for w in shape)
        raise ValueError(f"{name} must be an int32 tensor [{want}] on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t


def plan_step(cached: torch.Tensor, fresh: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
              taken: torch.Tensor, page_size: int, max_tokens: int) -> StepPlan:
    """Row starts, lengths, positions and slots of a step in which request b, with cached[b] tokens in the cache,
    brings fresh[b] more; block_table [B, width] gets the pages it takes from free_pages[taken ..], in the order of
    the requests. All int32 CUDA tensors. A request whose pages do not fit its row of block_table or what is left
    of the free list, whose rows would end behind max_tokens, or that would pass 2^31 - 1 tokens, is not served: it
    takes no page and its slots are -1. What one asks of the free list counts for those behind it: once it has run out, only
    requests that need no page are served. The caller goes on with the returned kv_len and taken; the same call again gives the same result."""
    _lib._need_cuda(cached, "cached")
    done = _lib.host.kv_plan(cached, fresh, block_table, free_pages, taken, page_size, max_tokens) \
        if page_size in PAGE_SIZES else None
    if done is not None:
        row_start, kv_len, positions, slots, taken, served = done
        return StepPlan(row_start, kv_len, positions, slots, taken, served)
    dev = cached.device
    _ints("cached", cached, (None,), dev)
    B = cached.shape[0]
    _ints("fresh", fresh, (B,), dev)
    _ints("block_table", block_table, (B, None), dev)
    _ints("free_pages", free_pages, (None,), dev)
    _ints("taken", taken, (1,), dev)
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    if not block_table.is_contiguous():
        raise ValueError("block_table is written in place: it must be contiguous")
    if B < 1 or B > 8192 or not 1 <= block_table.shape[1] <= INT_MAX or not 1 <= max_tokens <= INT_MAX:
        raise ValueError(f"plan_step: 1 to 8192 requests, a block_table of some width and max_tokens >= 1 wanted, both below "
                         f"2^31, got {B}, {block_table.shape[1]}, {max_tokens}")
    if free_pages.shape[0] > INT_MAX:
        raise ValueError(f"plan_step: fewer than 2^31 free pages wanted, got {free_pages.shape[0]}")
    return _plan_route(cached, fresh, block_table, free_pages, taken, page_size, max_tokens)


def _plan_route(cached, fresh, block_table, free_pages, taken, page_size, max_tokens):
    B, dev = cached.shape[0], cached.device
    cached, fresh, free_pages = cached.contiguous(), fresh.contiguous(), free_pages.contiguous()
    ints = torch.empty(2 * B + 2 + 2 * max_tokens, dtype=torch.int32, device=dev)
    row_start, kv_len, taken_out, positions, slots = ints.split((B + 1, B, 1, max_tokens, max_tokens))
    served = torch.empty(B, dtype=torch.bool, device=dev)
    a = _lib.KVPlanArgs(cached.data_ptr(), fresh.data_ptr(), block_table.data_ptr(), free_pages.data_ptr() or taken.data_ptr(),
                        taken.data_ptr(), row_start.data_ptr(), kv_len.data_ptr(), positions.data_ptr(),
                        slots.data_ptr(), taken_out.data_ptr(), served.data_ptr(), B, block_table.shape[1],
                        free_pages.shape[0], page_size, max_tokens)
    with _lib._on_device(dev):
        _lib.check(_lib.lib().b200lut_kv_plan(ctypes.byref(a), _lib._stream(cached)))
    return StepPlan(row_start, kv_len, positions, slots, taken_out, served)


class KVCache4:
    """n_pages pages of page_size tokens, n_kv_heads heads of head_dim elements (64, 128 or 256), for keys and values
    in `dtype`. A slot is page * page_size + offset. New caches hold zeros."""

    def __init__(self, n_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
        if n_pages < 1 or not 1 <= n_kv_heads <= 4096 or n_pages * page_size > 0x7fffffff:
            raise ValueError(f"n_pages >= 1, 1 to 4096 heads and fewer than 2^31 slots wanted, got {n_pages} pages of "
                             f"{page_size}, {n_kv_heads} heads")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("the cache must be on a CUDA device: this package computes on the GPU only")
        self.n_pages, self.n_kv_heads, self.head_dim = int(n_pages), int(n_kv_heads), int(head_dim)
        self.page_size, self.dtype = int(page_size), dtype
        codes = (2, n_pages, n_kv_heads, page_size * head_dim // 2)
        self._buffers = (*torch.zeros(codes, dtype=torch.uint8, device=device),
                         *torch.zeros((2, n_pages, n_kv_heads, page_size, 2), dtype=dtype, device=device))
        self.device = self.k_codes.device
        self._view = _lib.KVCacheView(self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.k_pairs.data_ptr(),
                                      self.v_pairs.data_ptr(), self.n_pages, self.page_size, self.n_kv_heads,
                                      self.head_dim, _lib.dtype_id(dtype))
        self._native = _lib.host.bind_cache(*self._buffers, self.n_pages, self.page_size, self.n_kv_heads, self.head_dim)

    # codes: uint8 [n_pages, n_kv_heads, page_size * head_dim / 2]; pairs (lo, hi): [n_pages, n_kv_heads, page_size, 2]
    k_codes = property(lambda self: self._buffers[0])
    v_codes = property(lambda self: self._buffers[1])
    k_pairs = property(lambda self: self._buffers[2])
    v_pairs = property(lambda self: self._buffers[3])

    def __reduce__(self):
        raise TypeError("a KVCache4 is bound to its device buffers: it is neither copied nor pickled")

    @property
    def nbytes(self) -> int:
        """Bytes on the device: (head_dim / 2 + 4) per token and head, for keys and for values."""
        return 2 * self.n_pages * self.page_size * self.n_kv_heads * (self.head_dim // 2 + 4)

    def _rows(self, name: str, x: torch.Tensor, heads: int) -> torch.Tensor:
        check_heads(name, x, heads, self.head_dim)
        if x.dtype != self.dtype or x.device != self.device:
            raise ValueError(f"{name} must be {self.dtype} on {self.device}, got {x.dtype} on {x.device}")
        return rows16(x)

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Rows k, v [tokens, n_kv_heads, head_dim] into `slots` (int32 [tokens], all different; negative: not
        written). A slot outside the cache is skipped and raises the device status (0x6100)."""
        if _lib.host.kv_write(self._native, k, v, slots):
            return
        k, v = self._rows("k", k, self.n_kv_heads), self._rows("v", v, self.n_kv_heads)
        T = k.shape[0]
        if v.shape[0] != T:
            raise ValueError(f"k has {T} tokens, v {v.shape[0]}")
        slots = _ints("slots", slots, (T,), self.device).contiguous()
        if T:
            with _lib._on_device(self.device):
                _lib.check(_lib.lib().b200lut_kv_write(ctypes.byref(self._view), k.data_ptr(), v.data_ptr(), k.stride(0),
                                                       k.stride(1), v.stride(0), v.stride(1), slots.data_ptr(), T,
                                                       _lib._stream(k)))

    def read(self, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [tokens, n_kv_heads, head_dim] that `slots` (int32 [tokens]) stand for, rounded to the
        cache's dtype; zeros for negative slots and for those outside the cache (device status 0x6100)."""
        done = _lib.host.kv_read(self._native, slots)
        if done is not None:
            return done
        if slots.dim() != 1:
            raise ValueError(f"slots must be an int32 tensor [*] on {self.device}, got {tuple(slots.shape)}")
        slots = _ints("slots", slots, (None,), self.device).contiguous()
        T = slots.shape[0]
        k, v = (torch.empty(T, self.n_kv_heads, self.head_dim, dtype=self.dtype, device=self.device) for _ in range(2))
        if T:
            with _lib._on_device(self.device):
                _lib.check(_lib.lib().b200lut_kv_read(ctypes.byref(self._view), k.data_ptr(), v.data_ptr(),
                                                      slots.data_ptr(), T, _lib._stream(k)))
        return k, v

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor,
               row_start: Optional[torch.Tensor] = None, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
               gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale q k^T) v of q [tokens, n_heads, head_dim] over the cache, [tokens, n_heads, head_dim].

        Rows row_start[b] .. row_start[b + 1] of q (int32 [B + 1]; without it one row per request) are the last tokens
        of request b, whose kv_len[b] tokens (int32 [B], the new ones written before) lie in the pages
        block_table[b] (int32 [B, width]). The row at position p sees the tokens j <= p; with a window those with
        j > p - window, and the first `sinks` tokens besides. Query head h reads key/value head
        h // (n_heads / n_kv_heads). scale: head_dim ** -0.5 unless given. gate: the result is multiplied by
        sigmoid(gate). out may be q or gate itself. Where nothing is visible the result is zero; rows that belong to no
        request are not written. A visible token on a page outside the cache counts as hidden and raises the device status
        (0x6200); pages that no row sees may be given away. The sums over tokens are fp32 and divided at the end."""
        done = _lib.host.attend(self._native, q, block_table, kv_len, row_start,
                                self.head_dim ** -0.5 if scale is None else scale, window, sinks, gate, out)
        if done is not None:
            return done
        if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % self.n_kv_heads:
            raise ValueError(f"q must be [tokens, a multiple of {self.n_kv_heads} heads, {self.head_dim}], got {tuple(q.shape)}")
        q = self._rows("q", q, q.shape[1])
        T, Hq, D = q.shape
        if out is not None:
            check_no_grad("out", out)
        if Hq // self.n_kv_heads > 64:
            raise ValueError(f"at most 64 query heads per key/value head, got {Hq // self.n_kv_heads}")
        _ints("block_table", block_table, (None, None), self.device)
        B, width = block_table.shape
        kv_len = _ints("kv_len", kv_len, (B,), self.device).contiguous()
        if row_start is not None:
            row_start = _ints("row_start", row_start, (B + 1,), self.device).contiguous()
        elif T != B:
            raise ValueError(f"without row_start there is one row per request: {T} rows, {B} requests")
        if window < 0 or sinks < 0 or not 1 <= width <= INT_MAX:
            raise ValueError("window and sinks must not be negative, and block_table needs some width, below 2^31")
        scale = D ** -0.5 if scale is None else float(scale)
        if not abs(scale) < 2.0 ** 127:              # 32 bits hold it, times log2(e) too
            raise ValueError(f"scale must be finite, below 2^127, got {scale}")
        if width > 1 and block_table.stride(1) != 1:
            block_table = block_table.contiguous()
        if gate is not None:
            if tuple(gate.shape) != (T, Hq, D):
                raise ValueError(f"gate must be [{T}, {Hq}, {D}], got {tuple(gate.shape)}")
            gate = self._rows("gate", gate, Hq)
        if out is None:
            out = torch.empty(T, Hq, D, dtype=self.dtype, device=self.device)
        to = None
        if tuple(out.shape) == (T, Hq, D) and out.dtype == self.dtype and out.device == self.device:
            to = rows16(out)
        if to is None or to.data_ptr() != out.data_ptr():
            raise ValueError(f"out must be [{T}, {Hq}, {D}] {self.dtype} on {self.device} with 16-byte rows")
        if T == 0 or B == 0:
            return out
        L = _lib.lib()
        with _lib._on_device(self.device):
            # a buffer of the current stream (of the capture's pool under capture): calls never share one
            ws = torch.empty(L.b200lut_attend_workspace_bytes(Hq, self.n_kv_heads, D, int(row_start is None)), dtype=torch.uint8, device=self.device)
            a = _lib.AttendArgs(ctypes.pointer(self._view), q.data_ptr(), _lib.ptr(gate), to.data_ptr(),
                                block_table.data_ptr(), kv_len.data_ptr(), _lib.ptr(row_start), q.stride(0), q.stride(1),
                                gate.stride(0) if gate is not None else 0, gate.stride(1) if gate is not None else 0,
                                to.stride(0), to.stride(1), block_table.stride(0), T, B, width, Hq, min(int(window), INT_MAX),
                                min(int(sinks), INT_MAX), scale)      # no cache holds more tokens
            _lib.check(L.b200lut_attend(ctypes.byref(a), ws.data_ptr(), ws.numel(), _lib._stream(q)))
        return out
