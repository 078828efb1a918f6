"""Rotary positions at the edges of their launch: more tokens than one row of
a grid takes."""
from __future__ import annotations

import pytest
import torch

import natten_mps_amd as na

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def test_more_blocks_than_one_grid_row():
    """2^30 tokens, 2^24 blocks of 64: a launch has fewer than 2^32 threads
    along x.  Parts of the result are those of the same tokens alone, at
    positions of their own."""
    tokens = 2 ** 30
    plan = na.RotaryPlan(2)
    x = torch.empty(1, tokens, 1, 2, dtype=torch.bfloat16, device=DEV)
    x.random_(-8, 9)
    out = na.rotary(x, plan)
    for lo in (0, 2 ** 29 - 500, tokens - 1000):
        part = slice(lo, lo + 1000)
        want = na.rotary(x[:, part], plan, torch.arange(lo, lo + 1000, device=DEV))
        assert torch.equal(out[:, part], want)
