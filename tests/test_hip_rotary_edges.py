"""Rotary positions at their edges: more tokens than one row of a grid takes,
forward-mode differentiation, far positions against the plan's own frequencies,
and sizes past 32 bits."""
from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch
from torch.autograd import forward_ad

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


def test_forward_mode():
    """A dual tensor's tangent turns as the tensor does; the paged calls have
    no gradients and refuse it."""
    plan = na.RotaryPlan(16)
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, dq, dk = (torch.randn(2, 5, h, 16, generator=g, device=DEV) for h in (4, 2, 4, 2))
    with forward_ad.dual_level():
        oq, ok = na.rotary_qk(forward_ad.make_dual(q, dq), k, plan)
        value, tangent = forward_ad.unpack_dual(oq)
        assert torch.equal(value, na.rotary(q, plan)) and torch.equal(tangent, na.rotary(dq, plan))
        assert torch.equal(ok, na.rotary(k, plan)) and not forward_ad.unpack_dual(ok).tangent.any()
        out = na.rotary(forward_ad.make_dual(k, dk), plan, torch.arange(5, device=DEV) + 3)
        want = na.rotary(dk, plan, torch.arange(5, device=DEV) + 3)
        assert torch.equal(forward_ad.unpack_dual(out).tangent, want)
        pages = torch.zeros(4, 4, 2, 16, device=DEV)
        table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
        lens = torch.full((2,), 5, dtype=torch.int32, device=DEV)
        with torch.no_grad(), pytest.raises(RuntimeError, match="dual tensors"):
            na.na1d_paged(forward_ad.make_dual(q, dq), pages, pages, table, lens)
        with torch.no_grad(), pytest.raises(RuntimeError, match="dual tensors"):
            na.na1d_paged_append(forward_ad.make_dual(k, dk), k, pages, pages.clone(), table, lens)


def test_far_positions_against_the_frequencies():
    """The angle is p f to 2^-65 |p| turns, f the plan's frequency itself;
    cosine and sine add two half steps of fp32 and 2e-9 of their series, and
    half a turn's last bit of the 32 that they see."""
    pi = Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
    plan = na.RotaryPlan(16)
    pos = [1, 10 ** 6 + 1, 2 ** 31 - 1, 2 ** 33 + 5, -(2 ** 36) - 3, 2 ** 40 + 77]
    x = torch.zeros(1, len(pos), 1, 16, device=DEV)
    x[..., :8] = 1  # out = (cos, sin)
    out = na.rotary(x, plan, torch.tensor(pos, device=DEV)).cpu().double()
    for i, n in enumerate(pos):
        for j, f in enumerate(plan.frequencies):
            angle = 2 * math.pi * float(n * Fraction(f) / (2 * pi) % 1)
            bound = 2 * 2.0 ** -24 + 2e-9 + 2 * math.pi * (2.0 ** -32 + abs(n) * 2.0 ** -65)
            assert abs(out[0, i, 0, j] - math.cos(angle)) <= bound
            assert abs(out[0, i, 0, 8 + j] - math.sin(angle)) <= bound


def test_sizes_past_32_bits_are_refused():
    """Views without memory of their own; nothing is launched or allocated."""
    plan = na.RotaryPlan(2)
    x = torch.zeros(1, 1, 1, 2, device=DEV)
    far = x.expand(1, 2 ** 32 + 5, 1, 2)
    with pytest.raises(NotImplementedError, match="2\\^31"):
        na.rotary(far, plan)
    pages = x.expand(2 ** 32 + 5, 1, 1, 2)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    with pytest.raises(NotImplementedError, match="2\\^31"):
        na.na1d_paged(x, pages, pages, table, lens)
    with pytest.raises(NotImplementedError, match="2\\^31"):
        na.na1d_paged(x, x, x, table.expand(1, 2 ** 32 + 5), lens)
    with pytest.raises(NotImplementedError, match="2\\^31"):
        na.na1d_paged_append(far, far, x.clone(), x.clone(), table, lens)
