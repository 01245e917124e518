"""The bounds that attention is held to reject a result that lacks a part, on the CPU."""
from __future__ import annotations

import pytest
import torch

from helpers_attention_tight import attend_tight, counted_values, counted_want


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("L", (70_001, 16_384, 1000))
@pytest.mark.parametrize("D", (64, 128, 256))
def test_a_missing_tile_is_outside_the_bound(D, L, dtype):
    # whichever 16 tokens are left out, one element or more moves by more than the bound
    v = counted_values(L, D)
    want, tol = counted_want(v, torch.tensor([L]), dtype)
    tiles = -(-L // 16)
    for tile in {0, 1, tiles // 3, tiles // 2, tiles - 2}:
        keep = torch.arange(L) // 16 != tile
        lacks = v[keep].sum(0) / keep.sum()                 # the part and its weight are lost
        kept = v[keep].sum(0) / L                           # the part is lost, its weight counted
        for got in (lacks, kept):
            assert ((got - want[0]).abs() / tol[0]).max() > 2, tile


def test_a_missing_block_is_outside_the_bound_of_rows_as_they_come():
    # an eighth of the tokens, of random rows and values: in the norm
    g = torch.Generator().manual_seed(0)
    L, D = 4096, 64
    k, v = (torch.randn(L, 1, D, generator=g).double() for _ in range(2))
    q = 1.5 * torch.randn(1, 2, D, generator=g).bfloat16()
    want, tol = attend_tight(q, k, v, torch.tensor([L - 1]), D ** -0.5)
    keep = torch.arange(L) >= L // 8
    less, _ = attend_tight(q, k[keep], v[keep], torch.tensor([keep.sum() - 1]), D ** -0.5)
    assert (less - want).norm() > tol.norm()
