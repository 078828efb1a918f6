"""Rotary positions on the GPU against the formula in float64: layouts, axes,
partly turned heads, odd sizes and strides, far positions, gradients, and use
on other streams and in graphs.

Tolerance.  A result is m (u c - v s) with c, s off by at most 2 half steps of
fp32 (angle, series, the factor m), two products and a sum of half a step
each: 4 * 2^-24 m (|u| + |v|) covers them.  Rounding to the output type adds
half a step of the value.
"""
from __future__ import annotations

import math

import pytest
import torch

import natten_mps_amd as na

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _coords(shape, plan, positions):
    sp = shape[1:-2]
    if positions is None:
        return torch.stack(torch.meshgrid(*(torch.arange(n) for n in sp), indexing="ij"), -1)[None]
    p = positions.cpu()
    p = p if plan.axes > 1 else p[..., None]
    return p if p.ndim == len(sp) + 2 else p[None]


def exact_turn(x, plan, positions=None, inverse=False):
    """(turned x, |u| + |v| of each element's pair) in float64 on the CPU."""
    x = x.detach().cpu().double()
    coords = _coords(x.shape, plan, positions)
    y, size = x.clone(), torch.zeros_like(x)
    n = plan.dim // plan.axes
    f = torch.tensor(plan.frequencies, dtype=torch.float64)
    for a in range(plan.axes):
        t = coords[..., a, None].double() * f * (-1 if inverse else 1)
        c, s = t.cos()[..., None, :], t.sin()[..., None, :]
        if plan.interleaved:
            one, two = slice(a * n, (a + 1) * n, 2), slice(a * n + 1, (a + 1) * n, 2)
        else:
            one, two = slice(a * n, a * n + n // 2), slice(a * n + n // 2, (a + 1) * n)
        u, v = x[..., one], x[..., two]
        y[..., one] = plan.magnitude * (u * c - v * s)
        y[..., two] = plan.magnitude * (u * s + v * c)
        size[..., one] = size[..., two] = plan.magnitude * (u.abs() + v.abs())
    return y, size


def check_turn(got, x, plan, positions=None, inverse=False, what=""):
    want, size = exact_turn(x, plan, positions, inverse)
    step = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    # float16 results below its normal range are off by half its smallest step
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bound = step * want.abs() * (1 + 2 ** -20) + (4 + 4 * step) * 2.0 ** -24 * size + tiny
    err = (got.detach().cpu().double() - want).abs()
    worst = (err - bound).max().item()
    assert worst <= 0, f"{what}: {err.max().item():.3g} off, {worst:.3g} past its bound"
    if plan.dim < x.shape[-1]:
        assert torch.equal(got[..., plan.dim:], x[..., plan.dim:].to(got.dtype)), f"{what}: copied dims"


def _randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(DEV, dtype)


CASES = [
    # shape, heads q/k, dim, plan, dtype
    ((2, 128), (4, 4), 32, dict(dim=32), torch.float32),
    ((1, 1), (1, 1), 2, dict(dim=2), torch.float32),
    ((3, 17), (6, 2), 64, dict(dim=64, scaling="ramp", factor=8, original_length=16), torch.bfloat16),
    ((2, 77), (5, 1), 80, dict(dim=20), torch.float16),               # 8-byte vectors
    ((2, 31), (3, 3), 48, dict(dim=38, interleaved=True), torch.bfloat16),   # single elements
    ((1, 9), (2, 1), 7, dict(dim=6), torch.float32),                  # odd head
    ((1, 9), (2, 1), 7, dict(dim=4, interleaved=True), torch.bfloat16),
    ((2, 7, 5), (4, 2), 32, dict(dim=32, axes=2, interleaved=True), torch.float16),
    ((2, 6, 11), (3, 3), 96, dict(dim=64, axes=2), torch.bfloat16),
    ((2, 3, 5, 4), (2, 2), 64, dict(dim=48, axes=3), torch.bfloat16),
    ((1, 4, 3, 9), (2, 1), 256, dict(dim=252, axes=3, interleaved=True), torch.float32),
    ((40, 300), (8, 2), 128, dict(dim=128, interleaved=True), torch.bfloat16),
    ((1, 20000), (1, 1), 32, dict(dim=16), torch.float16),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_rotary_qk_and_gradients(case):
    shape, heads, dim, plan, dtype = case
    plan = na.RotaryPlan(**plan)
    q, k = (_randn(i, *shape, h, dim, dtype=dtype).requires_grad_() for i, h in enumerate(heads))
    gq, gk = (_randn(7 + i, *shape, h, dim, dtype=dtype) for i, h in enumerate(heads))
    oq, ok = na.rotary_qk(q, k, plan)
    check_turn(oq, q, plan, what="q")
    check_turn(ok, k, plan, what="k")
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    check_turn(dq, gq, plan, inverse=True, what="dq")
    check_turn(dk, gk, plan, inverse=True, what="dk")
    assert torch.equal(na.rotary(k, plan), ok)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("shared", [True, False])
def test_explicit_positions(index, shared):
    plan = na.RotaryPlan(64)
    x = _randn(1, 3, 21, 4, 64)
    lead = () if shared else (3,)
    g = torch.Generator().manual_seed(5)
    p = torch.randint(0, 1 << 20, (*lead, 21), generator=g).to(DEV, index)
    check_turn(na.rotary(x, plan, p), x, plan, p)
    if not shared:
        check_turn(na.rotary(x, plan, p[:1]), x, plan, p[:1])
        strided = torch.stack((p, p + 1), -1)[..., 0]
        assert torch.equal(na.rotary(x, plan, strided), na.rotary(x, plan, p))


def test_explicit_positions_of_several_axes():
    plan = na.RotaryPlan(24, axes=3)
    x = _randn(2, 2, 13, 2, 32, dtype=torch.bfloat16)  # tokens of a packed grid
    g = torch.Generator().manual_seed(6)
    p = torch.randint(-50, 5000, (2, 13, 3), generator=g).to(DEV)
    check_turn(na.rotary(x, plan, p), x, plan, p)
    check_turn(na.rotary(x, plan, p[0]), x, plan, p[0])


def test_far_and_negative_positions():
    """Angles of positions past 2^32, against exact integer arithmetic on the
    frequency that the plan keeps."""
    plan = na.RotaryPlan(8)
    pos = [0, 1, -1, -4096, 10 ** 6, 2 ** 31 - 1, 2 ** 31, 2 ** 33 + 5, -(2 ** 40) - 3, 2 ** 62 + 12345]
    p = torch.tensor(pos, dtype=torch.int64, device=DEV)
    x = torch.zeros(1, len(pos), 1, 8, device=DEV)
    x[..., :4] = 1  # out = (cos, sin)
    out = na.rotary(x, plan, p).cpu().double()
    for i, n in enumerate(pos):
        for j, t in enumerate(plan._turns):
            turn = (n * t) % 2 ** 64 / 2.0 ** 64
            assert abs(out[0, i, 0, j] - math.cos(2 * math.pi * turn)) <= 2 * 2.0 ** -24 + 2e-9
            assert abs(out[0, i, 0, 4 + j] - math.sin(2 * math.pi * turn)) <= 2 * 2.0 ** -24 + 2e-9


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views(dtype):
    """q and k as views of a packed projection, an offset slice, crops of a
    grid, reversed axes, and an innermost stride that forces a copy."""
    plan = na.RotaryPlan(32, axes=2)
    qkv = _randn(3, 2, 9, 7, 3, 4, 32, dtype=dtype)
    q, k, _ = qkv.unbind(3)
    oq, ok = na.rotary_qk(q, k, plan)
    assert oq.is_contiguous()
    check_turn(oq, q, plan)
    check_turn(ok, k, plan)
    crop = _randn(4, 2, 12, 10, 4, 33, dtype=dtype)[:, 1:9, 2:9, :, 1:]  # elements at odd offsets
    check_turn(na.rotary(crop, plan), crop, plan)
    turned = _randn(5, 2, 7, 9, 4, 32, dtype=dtype).transpose(1, 2)
    check_turn(na.rotary(turned, plan), turned, plan)
    inner = _randn(6, 2, 9, 7, 32, 4, dtype=dtype).transpose(-1, -2)
    check_turn(na.rotary(inner, plan), inner, plan)
    shared = _randn(7, 1, 9, 7, 1, 32, dtype=dtype).expand(2, 9, 7, 4, 32)
    check_turn(na.rotary(shared, plan), shared, plan)


def test_gradients_of_sums_and_of_one_output():
    plan = na.RotaryPlan(16)
    q, k = _randn(1, 2, 5, 2, 16).requires_grad_(), _randn(2, 2, 5, 1, 16).requires_grad_()
    oq, ok = na.rotary_qk(q, k, plan)
    oq.sum().backward()  # an expanded gradient, and none for k
    check_turn(q.grad, torch.ones_like(q), plan, inverse=True)
    assert k.grad is None
    # a shared input takes the gradients of both uses
    x = _randn(3, 2, 5, 2, 16).requires_grad_()
    a, b = na.rotary_qk(x, x, plan)
    ga, gb = _randn(4, 2, 5, 2, 16), _randn(5, 2, 5, 2, 16)
    (gx,) = torch.autograd.grad((a, b), x, (ga, gb))
    one, two = (na.rotary(g, na.RotaryPlan(16, frequencies=[-f for f in plan.frequencies])) for g in (ga, gb))
    assert torch.allclose(gx, one + two, atol=1e-6)


def test_gradients_against_differences():
    """<g, f(x + h e) - f(x - h e)> / 2h along random directions: the map is
    linear, so the difference is exact up to rounding."""
    plan = na.RotaryPlan(12, axes=3, magnitude=1.25)
    x = _randn(1, 1, 2, 3, 4, 2, 16).requires_grad_()
    g, e = _randn(2, *x.shape), _randn(3, *x.shape)
    (gx,) = torch.autograd.grad(na.rotary(x, plan), x, g)
    with torch.no_grad():
        d = (na.rotary(x + e, plan) - na.rotary(x - e, plan)) / 2
    left, right = (g.double() * d.double()).sum().item(), (gx.double() * e.double()).sum().item()
    assert abs(left - right) <= 16 * 2.0 ** -24 * (g.abs() * (x.abs() + e.abs())).double().sum().item()


def test_second_derivative():
    plan = na.RotaryPlan(8)
    x = _randn(1, 1, 3, 1, 8).requires_grad_()
    g = _randn(2, 1, 3, 1, 8).requires_grad_()
    (gx,) = torch.autograd.grad(na.rotary(x, plan), x, g, create_graph=True)
    w = _randn(3, 1, 3, 1, 8)
    (gg,) = torch.autograd.grad(gx, g, w)
    assert torch.equal(gg, na.rotary(w, plan))


def test_nonfinite_stays_in_its_pair():
    plan = na.RotaryPlan(16)
    x = torch.ones(1, 4, 2, 16, device=DEV)
    x[0, 1, 0, 3] = math.nan
    x[0, 2, 1, 5] = math.inf
    bad = ~torch.isfinite(na.rotary(x, plan))
    want = torch.zeros_like(bad)
    want[0, 1, 0, 3] = want[0, 1, 0, 11] = True
    want[0, 2, 1, 5] = want[0, 2, 1, 13] = True
    assert torch.equal(bad, want)


def test_empty():
    plan = na.RotaryPlan(8)
    for shape in ((0, 4, 2, 8), (2, 0, 2, 8), (2, 4, 0, 8)):
        x = torch.zeros(shape, device=DEV)
        assert na.rotary(x, plan).shape == shape
    q, k = na.rotary_qk(torch.zeros(2, 4, 0, 8, device=DEV), _randn(1, 2, 4, 2, 8), plan)
    assert q.shape == (2, 4, 0, 8) and torch.equal(k, na.rotary(_randn(1, 2, 4, 2, 8), plan))


def test_refusals_on_the_device():
    plan = na.RotaryPlan(8)
    x = _randn(1, 2, 4, 2, 8)
    with pytest.raises(RuntimeError, match="same GPU|must live on"):
        na.rotary(x, plan, torch.arange(4))
    with pytest.raises(TypeError, match="mixed dtypes"):
        na.rotary_qk(x, x.half(), plan)
    with pytest.raises(TypeError, match="float32"):
        na.rotary(x.double(), plan)
    with pytest.raises(NotImplementedError, match="above 256"):
        na.rotary(_randn(1, 1, 2, 1, 264), plan)


def test_streams_and_graphs():
    plan = na.RotaryPlan(32)
    plan.table(DEV)
    x = _randn(1, 2, 50, 4, 32, dtype=torch.bfloat16)
    p = torch.arange(50, device=DEV)
    want = na.rotary(x, plan, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = na.rotary(x, plan, p)
    side.synchronize()
    assert torch.equal(got, want)
    # a captured forward and backward, replayed on changing inputs while an
    # eager graph of the same leaves lives
    leaf = x.clone().requires_grad_()
    alive = na.rotary(leaf, plan, p)
    g = _randn(2, *x.shape, dtype=torch.bfloat16)
    static = leaf.detach().clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = na.rotary(static, plan, p)
        (grad,) = torch.autograd.grad(out, static, g)
    for i in range(3):
        with torch.no_grad():
            static.copy_(_randn(10 + i, *x.shape, dtype=torch.bfloat16))
            p.copy_(torch.arange(50, device=DEV) * (i + 2))
        graph.replay()
        torch.cuda.synchronize()
        fresh = static.detach().clone().requires_grad_()
        eager = na.rotary(fresh, plan, p.clone())
        assert torch.equal(out, eager)
        assert torch.equal(grad, torch.autograd.grad(eager, fresh, g)[0])
    assert torch.equal(alive, want)


def test_table_is_not_made_during_capture():
    plan = na.RotaryPlan(32, base=777.0)
    x = _randn(1, 1, 4, 1, 32)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        with torch.cuda.graph(graph):
            na.rotary(x, plan)


@pytest.mark.parametrize("rank", [1, 2, 3])
def test_modules(rank):
    """A module with a plan attends with turned queries and keys, gradients
    included."""
    size, heads, dim = {1: (24,), 2: (9, 8), 3: (4, 6, 5)}[rank], 2, 24
    plan = na.RotaryPlan(2 * rank * 4, axes=rank)
    torch.manual_seed(0)
    m = getattr(na, f"NeighborhoodAttention{rank}D")(heads * dim, heads, 3, rotary=plan).to(DEV)
    x = _randn(1, 2, *size, heads * dim).requires_grad_()
    out = m(x)
    q, k, v = m.qkv(x).reshape(2, *size, 3, heads, dim).unbind(rank + 1)
    q, k = na.rotary_qk(q, k, plan)
    want = m.proj(getattr(na, f"na{rank}d")(q, k, v, kernel_size=3).reshape(2, *size, heads * dim))
    assert torch.equal(out, want)
    g = _randn(2, *out.shape)
    got = torch.autograd.grad(out, [x, *m.parameters()], g)
    ref = torch.autograd.grad(want, [x, *m.parameters()], g)
    for a, b in zip(got, ref):
        assert torch.allclose(a, b, atol=1e-5, rtol=1e-5)
