"""Rotary positions and the paged cache under the program around them, without
a GPU: forward-mode differentiation, traces, how well turns hold a frequency,
the bookkeeping of many pages, inputs that do not fit what was reserved,
modules from before there were plans, and limits."""
from __future__ import annotations

import ctypes
import math
import random
import time
from fractions import Fraction

import pytest
import torch
from torch.autograd import forward_ad

import natten_mps_amd as na
from natten_mps_amd import positions as positions_module
from natten_mps_amd._core import _lib
from test_rotary_cpu import _cache, _cache_args, _held, _paged


def turn(x, plan, positions, inverse):
    """The formula for one axis of pairs (j, j + n / 2), in torch operations."""
    f = torch.tensor(plan.frequencies, dtype=x.dtype)
    at = torch.arange(x.shape[1]) if positions is None else positions
    t = (at[..., None] * f * (-1 if inverse else 1))[..., None, :]
    u, v = x[..., :plan.dim].chunk(2, -1)
    turned = torch.cat((u * t.cos() - v * t.sin(), u * t.sin() + v * t.cos()), -1) * plan.magnitude
    return torch.cat((turned, x[..., plan.dim:]), -1)


@pytest.fixture
def formula(monkeypatch):
    """The formula in the kernels' place: as they do, it sees no gradients."""
    def hook(q, k, plan, positions, inverse):
        q, k = (None if t is None else forward_ad.unpack_dual(t).primal.detach() for t in (q, k))
        return [None if t is None else turn(t, plan, positions, inverse) for t in (q, k)]

    monkeypatch.setattr(positions_module, "_hook", lambda: hook)


@pytest.mark.parametrize("explicit", [False, True])
def test_forward_mode_carries_the_tangent(formula, explicit):
    plan = na.RotaryPlan(8, magnitude=1.5)
    g = torch.Generator().manual_seed(1)
    q, k, dq, dk = (torch.randn(2, 5, h, 10, generator=g, dtype=torch.float64) for h in (3, 2, 3, 2))
    pos = torch.arange(5) + 7 if explicit else None
    with forward_ad.dual_level():
        for tangents in ((dq, dk), (dq, None), (None, dk)):
            duals = [x if d is None else forward_ad.make_dual(x, d) for x, d in zip((q, k), tangents)]
            out = na.rotary_qk(*duals, plan, pos)
            for o, x, d in zip(out, (q, k), tangents):
                value, tangent = forward_ad.unpack_dual(o)
                assert torch.equal(value, turn(x, plan, pos, False))
                assert torch.equal(tangent, torch.zeros_like(x) if d is None else turn(d, plan, pos, False))
        with torch.no_grad():
            tangent = forward_ad.unpack_dual(na.rotary(forward_ad.make_dual(q, dq), plan, pos)).tangent
        assert torch.equal(tangent, turn(dq, plan, pos, False))
    assert torch.autograd.gradcheck(lambda a, b: na.rotary_qk(a, b, plan, pos),
                                    (q.requires_grad_(), k.requires_grad_()), check_forward_ad=True,
                                    check_batched_grad=False)


@pytest.mark.parametrize("name", ["key", "value", "key_pages", "value_pages", "query"])
def test_paged_calls_refuse_tangents(name):
    a = _cache_args()
    a["query"] = torch.zeros(2, 3, 4, 8)
    with forward_ad.dual_level():
        a[name] = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
        with torch.no_grad(), pytest.raises(RuntimeError, match="dual tensors"):
            na.na1d_paged_append(**a)
        if name in ("key", "value"):
            return
        del a["key"], a["value"]
        with pytest.raises(RuntimeError, match="dual tensors"):
            na.na1d_paged(**a)


def test_tables_of_a_trace_are_not_kept():
    """A table made under fake tensors, or inside a compiled function, is the
    trace's own: real calls of this and of an equal plan get real ones."""
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode

    def plan():
        return na.RotaryPlan(8, base=123.0)

    p = plan()
    with FakeTensorMode():
        assert isinstance(p.table("cpu"), FakeTensor)
    for x in (p, plan()):
        assert type(x.table("cpu")) is torch.Tensor
        assert x.table("cpu").tolist() == list(p._turns)
    p = na.RotaryPlan(8, base=124.0)
    seen = set(positions_module._TABLES)
    out = torch.compile(lambda x: x + p.table("cpu"), backend="eager")(torch.zeros(4, dtype=torch.int64))
    assert out.tolist() == list(p._turns)
    assert set(positions_module._TABLES) == seen and not p._tables
    assert p.table("cpu").tolist() == list(p._turns)
    with FakeTensorMode():
        assert type(p.table("cpu")) is torch.Tensor  # one that is there serves


# 100 digits: 2^-332
PI = Fraction("3.1415926535897932384626433832795028841971693993751058209749445923078164062862089986280348253421170679")


@pytest.mark.parametrize("sign", [1, -1])
def test_turns_are_the_nearest_fractions(sign):
    """Each turn is f / (2 pi) modulo 1 to half of 2^-64, f the float as it
    is: whatever its size, as far as the digits of pi here reach."""
    freqs = [1.0, 0.25, 7.0, 1e-9, 5e-324, 2 * math.pi, 100.0, 3.0, 1e20, 2.0 ** 100, 10000.0 ** (-2 / 64), 1 / 3, 0.0,
             1e-300, 2.0 ** 64 / math.pi, 123456.789]
    p = na.RotaryPlan(32, frequencies=[sign * f for f in freqs])
    for f, t in zip(p.frequencies, p._turns):
        assert -2 ** 63 <= t < 2 ** 63
        gap = (Fraction(t, 2 ** 64) - Fraction(f) / (2 * PI)) % 1
        assert min(gap, 1 - gap) <= Fraction(1, 2 ** 65) + Fraction(1, 2 ** 150), f
    assert len(na.RotaryPlan(2, frequencies=[1.7e308])._turns) == 1


def test_cache_follows_any_order_of_calls():
    """The device's tables and lengths against the host's lists."""
    rng = random.Random(3)
    c = _cache(num_pages=40, batch=4, max_pages=12)
    for _ in range(300):
        op = rng.random()
        if op < 0.6:
            try:
                c.reserve([rng.choice((0, 0, 1, 1, 2, 9)) for _ in range(4)])
            except RuntimeError:
                c.release(rng.randrange(4))
        elif op < 0.8:
            c.trim(rng.choice((1, 3, 8)), rng.choice((1, 2)))
        else:
            c.release(rng.randrange(4))
        _held(c)
        assert c.block_table.tolist() == [t + [-1] * (12 - len(t)) for t in c._tables]
        assert c.seq_lens.tolist() == c.lengths and c.new_lens.tolist() == c._new


def test_cache_of_many_pages_is_quick_to_update():
    """What a step costs goes by the sequences and the pages that change, not
    by the table's size."""
    c = _cache(num_pages=1 << 16, page_size=1, batch=256, max_pages=1 << 13, head_dim=1, num_kv_heads=1)
    c.reserve(8)
    t = time.perf_counter()
    for _ in range(5):
        c.reserve(1)
    assert (time.perf_counter() - t) / 5 < 0.1
    t = time.perf_counter()
    c.release(7)
    assert time.perf_counter() - t < 0.1


def test_module_refuses_fewer_tokens_than_reserved():
    """They would be taken for the last ones of each sequence, and the slots
    before them would hold what was there."""
    c = _cache()
    c.reserve([5, 0, 4])
    assert c.new_tokens == 5
    m = na.NeighborhoodAttention1D(16, 2, 3, is_causal=True)
    with torch.no_grad(), pytest.raises(ValueError, match="5 new tokens of a sequence reserved, x holds 4"):
        m(torch.zeros(3, 4, 16), cache=c.layer(0))


def test_module_saved_before_plans(pure_backend):
    """A module saved whole by an earlier version has no ``rotary`` of its
    own: it runs as it did."""
    m = na.NeighborhoodAttention1D(16, 2, 3)
    x = torch.randn(2, 9, 16)
    want = m(x)
    state = m.__getstate__() if hasattr(m, "__getstate__") else m.__dict__.copy()
    old = na.NeighborhoodAttention1D.__new__(na.NeighborhoodAttention1D)
    old.__setstate__({n: v for n, v in state.items() if n != "rotary"})
    assert torch.equal(old(x), want)


def test_rows_past_31_bits_are_refused():
    """The elements of a token's row are counted in 32 bits."""
    lib, lay, d = _lib.load(), ctypes.byref(_lib.Layout()), ctypes.c_void_p(16)
    p = _paged(batch=1, tokens=1, heads_q=2 ** 24, dim_v=128)
    rc = lib.natten_hip_paged_forward(ctypes.byref(p), d, d, None, d, lay, d, d, d, lay, d, lay, None, 0, None)
    assert rc == 2 and "heads x dim_v" in lib.natten_hip_last_error().decode()
    assert lib.natten_hip_paged_workspace(ctypes.byref(p)) == -1
    assert lib.natten_hip_paged_workspace(ctypes.byref(_paged(batch=1, tokens=1, heads_q=2 ** 23, dim_v=128))) >= 0
