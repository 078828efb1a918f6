"""Attention over a paged cache where its arithmetic has edges: values that are
not finite, beside rows that do not attend to them and in long runs of keys,
windows of any length beside tokens before the sequence, probabilities far
below the largest one, instances of the kernels that the ordinary cases do not
reach, and more tiles than a row of a grid takes.  Tolerances are those of
``test_hip_paged``."""
from __future__ import annotations

import math
import time

import pytest
import torch

import natten_mps_amd as na
from test_hip_paged import BF, DEV, F32, FP, Problem, check

pytestmark = pytest.mark.gpu


def _at(p, seq, pos):
    """Page and slot of a position."""
    return p.table[seq, pos // p.page].long(), pos % p.page


def exact_rows(p, seq, tokens, kernel=None, dilation=1):
    """(out, lse, sum of p |v| over finite values, largest score error per
    unit 2^-24) of some of a sequence's new tokens, in float64 on the CPU.
    A value that is not finite comes out as itself wherever a key that the
    token attends to holds it."""
    n, length = p.news[seq].item(), p.lens[seq].item()
    have = torch.arange(length)
    pages = p.table[seq].cpu().long()[have // p.page]
    have = have[pages >= 0]
    pages = pages[pages >= 0]
    k, v = (t.cpu()[pages, have % p.page].double() for t in (p.kp, p.vp))
    H, D = p.q.shape[2:]
    rep = H // p.hkv
    res = []
    for i in tokens:
        back = length - n + i - have
        ok = back >= 0
        if kernel is not None:
            ok &= (back % dilation == 0) & (back < kernel * dilation)
        ki, vi = k[ok].repeat_interleave(rep, 1), v[ok].repeat_interleave(rep, 1)
        q = p.q[seq, i].cpu().double()
        s = (ki * q).sum(-1) * D ** -0.5
        w = s.softmax(0)[..., None] if len(s) else torch.zeros(0, H, 1, dtype=torch.float64)
        res.append(((w * vi).sum(0), s.logsumexp(0) if len(s) else torch.full((H,), -math.inf, dtype=torch.float64),
                    (w * torch.where(vi.isfinite(), vi.abs(), 0)).sum(0),
                    (ki.abs() * q.abs()).sum(-1).amax(0) * D ** -0.5 if len(s) else torch.zeros(H, dtype=torch.float64)))
    return [torch.stack(x) for x in zip(*res)]


def check_rows(got, p, seq, tokens, kernel=None, dilation=1, slack=0.0, lse_slack=0.0, what=""):
    """The bound of ``test_hip_paged.check`` at finite results, the others
    exactly."""
    want, wlse, mag, err = exact_rows(p, seq, tokens, kernel, dilation)
    out, lse = (t[seq, list(tokens)].cpu() for t in got)
    step = torch.finfo(out.dtype).eps / 2
    n = max(p.lens[seq].item(), 1)
    sums = (8 + n ** 0.5) * 2.0 ** -24
    delta = (p.q.shape[-1] + 4) * 2.0 ** -24 * err
    probs = 0.0 if out.dtype == F32 else step
    fin = want.isfinite()
    bound = step * want.abs() + (probs + sums + 2 * delta[..., None]) * mag * 1.01 + slack
    bound += torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
    diff = (out.double() - want).abs()
    assert torch.isfinite(out[fin]).all(), f"{what}: {(~torch.isfinite(out[fin])).sum()} results are not finite"
    worst = (diff - bound)[fin].max().item() if fin.any() else 0.0
    assert worst <= 0, f"{what}: {diff[fin].max().item():.3g} off, {worst:.3g} past its bound"
    assert torch.equal(out.double()[~fin].nan_to_num(nan=7.0), want[~fin].nan_to_num(nan=7.0)), f"{what}: not finite"
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (out[empty] == 0).all(), f"{what}: rows without keys"
    d = (lse.double() - wlse)[~empty].abs() - (delta + sums + 4 * 2.0 ** -24 * (1 + wlse.abs()) + lse_slack)[~empty]
    assert d.numel() == 0 or d.max().item() <= 0, f"{what}: lse"


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("new, length, hq, hkv", [
    (5, 5890, 4, 2),     # parts of 256 keys, two keys in the last: few rows
    (70, 65537, 2, 1),   # parts of 2048 keys, one key in the last: many rows
])
def test_rows_without_a_key_in_a_part(new, length, hq, hkv, bad, dtype):
    """Keys are cut and the last part holds the newest keys alone: a value
    there that is not finite stays with the tokens that attend to it."""
    p = Problem([(new, length)], hq, hkv, 32 if hkv == 1 else 64, 64, dtype)
    p.vp[_at(p, 0, length - 1)] = bad
    got = p.run()
    check_rows(got, p, 0, sorted({0, 1, new // 2, new - 2, new - 1}))
    assert torch.isfinite(got[0][0, :new - 1]).all()


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("new, hq", [(8, 2), (8, 8), (70, 4)])
def test_rows_without_a_key_beside_others(new, hq, dtype):
    """Tokens whose pages are all absent are empty, whatever the values of
    the tokens beside them hold."""
    p = Problem([(new, 200)], hq, 2, 64, 4, dtype)
    first = 200 - new
    gone = [j // 4 for j in range(first - 1, 196)]
    p.table[0, gone] = -1
    for j, bad in ((196, math.inf), (198, math.nan), (199, -math.inf)):
        p.vp[_at(p, 0, j)[0], j % 4, :, 3:] = bad
    got = p.run(2)
    check_rows(got, p, 0, range(new), 2)
    assert (got[1][0, :196 - first] == -math.inf).all()


def _seconds(fn, n=3):
    fn()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(n):
        fn()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) / n


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new, length, kernel", [(4, 2000, None), (512, 2000, None), (512, 2000, 600)])
def test_nonfinite_values_cost_a_few_walks(new, length, kernel, dtype):
    """A value at an early key that is not finite, seen by all or by some
    rows of a tile: the rows that are summed again cost a few more walks over
    the keys, not a dot product for each head dim."""
    p = Problem([(new, length)], 4, 2, 128, 16, dtype)
    plain = _seconds(lambda: p.run(kernel))
    p.vp[_at(p, 0, length - new - 100)] = math.inf
    p.vp[_at(p, 0, length - 1)] = math.nan
    got = p.run(kernel)
    check_rows(got, p, 0, sorted({0, 1, new // 2, new - 1}), kernel)
    assert _seconds(lambda: p.run(kernel), 1) <= 30 * plain + 1e-3


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("new, length, hq, hkv, dim, kernel, dil", [
    (6, 90, 4, 2, 64, 30, 1), (6, 90, 4, 2, 128, 30, 2), (90, 200, 4, 2, 64, 40, 1), (90, 200, 4, 2, 128, 40, 1),
    (90, 200, 4, 2, 96, None, 1), (90, 200, 4, 2, 32, 11, 3), (40, 5000, 2, 2, 64, 3000, 1), (90, 5000, 2, 1, 64, 3000, 1),
])
def test_nonfinite_values_key_by_key(new, length, hq, hkv, dim, kernel, dil, dtype):
    """Infinities of both signs and NaN at keys that some tokens attend to
    and others do not, in dims of their own and in shared ones."""
    p = Problem([(new, length), (3, 40)], hq, hkv, dim, 16, dtype)
    for j, d, bad in ((length - 1, 0, math.inf), (length - new, 1, -math.inf), (length - new // 2, 2, math.nan),
                      (length - new // 3, 3, math.inf), (length - 2, 3, -math.inf), (length - new // 2, 17, -math.inf),
                      (length - new // 3, 17, -math.inf), (0, dim - 1, math.inf)):
        pg, slot = _at(p, 0, j)
        p.vp[pg, slot, 0, d] = bad
    got = p.run(kernel, dil)
    check_rows(got, p, 0, range(new) if length < 1000 else range(0, new, 7), kernel, dil)
    check_rows(got, p, 1, range(3), kernel, dil)
    assert all(torch.equal(a.nan_to_num(nan=9.0), b.nan_to_num(nan=9.0)) for a, b in zip(p.run(kernel, dil), got))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hq, hkv, dim, dil", [(2, 2, 64, 1), (8, 2, 64, 1), (2, 2, 128, 2), (8, 2, 32, 2), (2, 1, 20, 1)])
@pytest.mark.parametrize("kernel", [2 ** 31 - 1, 2 ** 31 - 5])
def test_window_past_all_with_tokens_before_the_sequence(hq, hkv, dim, dil, kernel, dtype):
    """A window of any length over a sequence shorter than its new tokens:
    the tokens before position 0 are empty, the others see what there is."""
    p = Problem([(40, 40), (40, 40)], hq, hkv, dim, 16, dtype)
    p.lens = torch.tensor([30, 1], dtype=torch.int32, device=DEV)
    check(p.run(kernel, dil), p, kernel, dil)


@pytest.mark.parametrize("new, dim", [(1, 32), (1, 64), (1, 128), (70, 32), (70, 64), (70, 128)])
def test_probabilities_far_below_the_largest(new, dim):
    """One early key takes nearly all of the weight, thousands hold 2^-25 of
    it each.  A probability in fp16 is off by half a step, below its normal
    range by 2^-25 over the factor 2^7 that it carries: 2^-32 of the largest
    one and of the largest value for each key.  The sum of n positive terms in
    fp32 is off by at most n half steps, n 2^-24 of itself; the module's
    sqrt(n) holds for errors of either sign, but here each small term lies
    below half a step of the sum that holds the large one, so all are lost
    the same way.  lse is off by as much (the logarithm's slope is 1 over the
    sum)."""
    B, hkv, length = 64, 8, 4096
    p = Problem([(new, length)], hkv, hkv, dim, 64, FP)
    g = torch.Generator().manual_seed(1)
    p.table = p.table.expand(B, -1).contiguous()  # one sequence's pages, read by all
    p.lens, p.news = p.lens.expand(B).contiguous(), p.news.expand(B).contiguous()
    p.q = (torch.randn(B, new, hkv, dim, generator=g) * 0.01).to(DEV, FP)
    p.q[..., 0] = 8.0
    p.kp = (torch.randn(p.kp.shape, generator=g) * 0.01).to(DEV, FP)
    p.kp[..., 0] = 0.0
    pg, slot = _at(p, 0, 3)
    p.kp[pg, slot, :, 0] = 25.4 * math.log(2) * dim ** 0.5 / 8
    p.vp = (64 + torch.randn(p.vp.shape, generator=g)).to(DEV, FP)
    p.vp[pg, slot] = 0.0
    got = p.run()
    for seq in (0, B - 1):
        check_rows(got, p, seq, sorted({0, new - 1}), slack=length * 2.0 ** -32 * p.vp.abs().max().item(),
                   lse_slack=length * 2.0 ** -24)


# rows (new, length), heads q/kv, dim, page, kernel, dilation, dtype
INSTANCES = {
    "chunk_dim96": ([(129, 200), (40, 300)], 4, 2, 96, 16, None, 1, BF),
    "chunk_dim96_window": ([(129, 200), (40, 300)], 4, 2, 96, 8, 37, 1, FP),
    "chunk_dim96_cut": ([(40, 4500)], 2, 1, 96, 64, None, 1, FP),
    "chunk_dim32": ([(150, 150), (97, 400)], 4, 2, 32, 16, None, 1, BF),
    "chunk_dim32_window": ([(150, 150), (97, 400)], 4, 1, 32, 5, 50, 1, FP),
    "chunk_dim32_cut": ([(70, 4500)], 2, 1, 32, 64, 4200, 1, BF),
    "few_dim64_four": ([(5, 700), (4, 300)], 8, 1, 64, 64, None, 1, FP),
    "few_dim64_four_cut": ([(5, 9000), (5, 31)], 8, 1, 64, 64, None, 1, FP),
    "few_dim64_four_bf16": ([(60, 90), (33, 200)], 2, 2, 64, 16, 41, 1, BF),
    "few_dim64_two": ([(5, 700), (4, 300)], 8, 2, 64, 16, None, 1, BF),
    "few_dim96_two": ([(5, 700), (4, 300)], 8, 2, 96, 16, None, 1, BF),
    "few_dim96_two_window": ([(30, 200), (17, 40)], 2, 2, 96, 16, 21, 1, FP),
    "few_dim128_two": ([(5, 700), (4, 300)], 8, 2, 128, 16, None, 1, FP),
    "few_dim128_two_cut": ([(5, 9000), (2, 5)], 8, 2, 128, 32, None, 1, BF),
    "few_fp32_dim128_one": ([(2, 300), (1, 77)], 8, 2, 128, 16, None, 1, F32),
    "few_fp32_dim128_one_cut": ([(2, 5000), (1, 77)], 4, 2, 128, 16, None, 1, F32),
    "few_fp32_dim64_one": ([(1, 700), (1, 64)], 16, 2, 64, 16, 300, 1, F32),
    "few_fp32_dim64_two": ([(5, 700), (4, 300)], 8, 2, 64, 16, None, 1, F32),
    "few_fp32_dim96_one": ([(2, 300), (1, 77)], 8, 2, 96, 24, None, 1, F32),
    "few_fp32_dim32_one": ([(2, 300), (1, 77)], 8, 2, 32, 16, None, 1, F32),
}


@pytest.mark.parametrize("name", INSTANCES)
def test_instances_against_float64(name):
    rows, hq, hkv, dim, page, kernel, dil, dtype = INSTANCES[name]
    p = Problem(rows, hq, hkv, dim, page, dtype, seed=len(name))
    check(p.run(kernel, dil), p, kernel, dil, what=name)


@pytest.mark.parametrize("tokens, dim, kernel, dil", [
    (2 ** 26, 8, 1, 1),        # 2^24 tiles of four rows
    (2 ** 24, 32, 2, 2 ** 24),  # a dilation that leaves each token alone: 2^24 tiles
])
def test_more_tiles_than_one_grid_row(tokens, dim, kernel, dil):
    """A launch has fewer than 2^32 threads along x.  Each token sees itself
    alone here: its own value comes out, and its logit as lse."""
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(1, tokens, 1, dim, generator=g, device=DEV, dtype=BF) for _ in range(3))
    pages = tokens // 64
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([tokens], dtype=torch.int32, device=DEV)
    out, lse = na.na1d_paged(q, k.view(pages, 64, 1, dim), v.view(pages, 64, 1, dim), table, lens, kernel, dil,
                             return_lse=True)
    assert torch.equal(out, v)
    for part in (slice(0, 4096), slice(tokens // 2 - 99, tokens // 2 + 99), slice(tokens - 4096, None)):
        s = (q[:, part].float() * k[:, part].float()).sum(-1) * dim ** -0.5
        assert torch.allclose(lse[:, part], s, atol=1e-5, rtol=1e-5)
