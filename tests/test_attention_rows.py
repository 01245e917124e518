"""Rows of heads as the attention side's fronts hand them on, on the CPU."""
from __future__ import annotations

import torch

from conftest import load_pkg

pkg = load_pkg()


def test_rows_of_one_token_or_one_head_have_any_stride():
    # a single token's stride is nobody's: no copy, and nothing the C entries refuse
    rows16 = pkg.rotary.rows16
    wide = torch.arange(5 * 516, dtype=torch.float32).bfloat16().view(5, 516)
    many = wide[:, :512].unflatten(1, (4, 128))
    for x, copied in ((many[:1], False), (many, True), (many[2:3], False), (torch.zeros(1, 1, 130)[..., :128].bfloat16(), False),
                      (torch.zeros(3, 1, 136).bfloat16()[..., :128], False), (torch.zeros(3, 1, 130).bfloat16()[..., :128], True),
                      (torch.zeros(1, 2, 130).bfloat16()[..., :128], True), (torch.zeros(1, 1, 200).bfloat16()[..., 1:129], True),
                      (wide.flatten()[1:513].view(1, 4, 128), True), (many[:0], True)):
        y = rows16(x)
        assert torch.equal(y, x) and y.stride(2) == 1 and y.stride(0) % 8 == 0 and y.stride(1) % 8 == 0
        assert x.numel() == 0 or y.data_ptr() % 16 == 0
        assert x.numel() == 0 or (y.data_ptr() != x.data_ptr()) == (copied or x.data_ptr() % 16 != 0)
