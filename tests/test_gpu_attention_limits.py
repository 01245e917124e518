"""The attention side at the ends of what its arguments can say, on the GPU."""
from __future__ import annotations

import pytest
import torch

from conftest import load_pkg

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
