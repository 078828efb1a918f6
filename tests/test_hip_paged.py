"""Attention over a paged cache, and appending to it, on the GPU against
float64: head layouts, windows, dilations, lengths from none to long, odd
pages, strides, absent pages, non-finite values outside of windows, streams,
graphs, and a run of append and attention against na1d.

Tolerance of attention.  A score is a sum of D products in fp32, off by at
most (D + 2) 2^-24 of its sum of magnitudes, delta after scaling; e^s is then
off by delta of itself, in numerator and denominator.  16-bit kernels round
each probability once for the product with v (half a step of the type, and of
the product of fp32 sums of n terms n 2^-24 at most, sqrt(n) in practice; the
parts add theirs).  The result rounds once.
"""
from __future__ import annotations

import math

import pytest
import torch

import natten_mps_amd as na
from test_hip_rotary import check_turn, exact_turn

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(DEV, dtype)


class Problem:
    """Sequences of (new, length) over shuffled pages; entries past a
    sequence's end name no page."""

    def __init__(self, rows, hq, hkv, dim, page, dtype, dim_v=None, tokens=None, seed=0, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.page, self.hkv = rows, page, hkv
        self.tokens = max(n for n, _ in rows) if tokens is None else tokens
        dim_v = dim if dim_v is None else dim_v
        per = [-(-max(length, 0) // page) for _, length in rows]
        pages = sum(per) + spare
        order = torch.randperm(pages, generator=g).tolist()
        wide = max(max(per), 1)
        table = [[order.pop() for _ in range(n)] + [-1] * (wide - n) for n in per]
        self.table = torch.tensor(table, dtype=torch.int32, device=DEV)
        self.lens = torch.tensor([n for _, n in rows], dtype=torch.int32, device=DEV)
        self.news = torch.tensor([n for n, _ in rows], dtype=torch.int32, device=DEV)
        self.kp = _randn(seed + 1, pages, page, hkv, dim, dtype=dtype)
        self.vp = _randn(seed + 2, pages, page, hkv, dim_v, dtype=dtype)
        self.q = _randn(seed + 3, len(rows), self.tokens, hq, dim, dtype=dtype)

    def run(self, kernel=None, dilation=1, **kw):
        return na.na1d_paged(self.q, self.kp, self.vp, self.table, self.lens, kernel, dilation, new_lens=self.news,
                             return_lse=True, **kw)


def exact(p, kernel=None, dilation=1, scale=None):
    """(out, lse, sum of p |v|, largest score error per unit 2^-24) on the
    CPU in float64; keys on absent pages are left out."""
    q, kp, vp, table = p.q.cpu().double(), p.kp.cpu().double(), p.vp.cpu().double(), p.table.cpu().long()
    B, L, H, D = q.shape
    rep = H // p.hkv
    scale = D ** -0.5 if scale is None else scale
    out, mag = torch.zeros(B, L, H, vp.shape[-1], dtype=torch.float64), None
    mag = torch.zeros_like(out)
    lse = torch.full((B, L, H), -math.inf, dtype=torch.float64)
    err = torch.zeros(B, L, H, dtype=torch.float64)
    cap = table.shape[1] * p.page
    for b, (n, length) in enumerate(zip(p.news.tolist(), p.lens.tolist())):
        n = min(max(n, 0), L)
        length = max(length, 0)
        have = torch.arange(min(length, cap))
        pg = table[b, have // p.page]
        have = have[(pg >= 0) & (pg < kp.shape[0])]
        pg = table[b, have // p.page]
        k, v = kp[pg, have % p.page], vp[pg, have % p.page]  # [n, Hkv, D]
        for i in range(n):
            pos = length - n + i
            back = pos - have
            ok = back >= 0
            if kernel is not None:
                ok &= (back % dilation == 0) & (back < kernel * dilation)
            if not bool(ok.any()):
                continue
            ki, vi = k[ok].repeat_interleave(rep, 1), v[ok].repeat_interleave(rep, 1)
            s = (ki * q[b, i]).sum(-1) * scale  # [keys, H]
            w = s.softmax(0)
            out[b, i] = (w[..., None] * vi).sum(0)
            mag[b, i] = (w[..., None] * vi.abs()).sum(0)
            lse[b, i] = s.logsumexp(0)
            err[b, i] = ((ki.abs() * q[b, i].abs()).sum(-1) * abs(scale)).amax(0)
    return out, lse, mag, err


def check(got, p, kernel=None, dilation=1, scale=None, what=""):
    out, lse = (t.cpu() for t in got)
    want, wlse, mag, err = exact(p, kernel, dilation, scale)
    assert lse.dtype == torch.float32 and out.shape == want.shape and out.dtype == p.q.dtype
    D = p.q.shape[-1]
    step = torch.finfo(out.dtype).eps / 2
    n = max(max(p.lens.tolist()), 1)
    sums = (8 + n ** 0.5) * 2.0 ** -24
    delta = (D + 4) * 2.0 ** -24 * err
    probs = 0.0 if out.dtype == torch.float32 else step
    bound = step * want.abs() + (probs + sums + 2 * delta[..., None]) * mag * 1.01
    bound += torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
    diff = (out.double() - want).abs()
    worst = (diff - bound).max().item() if diff.numel() else 0.0
    assert worst <= 0, f"{what}: out {diff.max().item():.3g} off, {worst:.3g} past its bound"
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty), f"{what}: rows without keys"
    assert (out[empty] == 0).all(), f"{what}: rows without keys hold zeros"
    d = (lse.double() - wlse)[~empty].abs() - (delta + sums + 4 * 2.0 ** -24 * (1 + wlse.abs()))[~empty]
    assert d.numel() == 0 or d.max().item() <= 0, f"{what}: lse {d.max().item():.3g} past its bound"


BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32

# rows (new, length), heads q/kv, dim, page, kernel, dilation, dtype
CASES = {
    "one": ([(1, 1)], 1, 1, 32, 16, None, 1, BF),
    "tokens": ([(1, 5), (1, 64), (1, 65), (1, 200)], 8, 2, 64, 16, None, 1, BF),
    "tokens_fp32": ([(1, 5), (1, 64), (1, 65), (1, 200)], 8, 2, 64, 16, None, 1, F32),
    "tokens_window": ([(1, 3), (1, 33), (1, 500)], 4, 2, 128, 16, 33, 4, FP),
    "tokens_mqa": ([(1, 130), (1, 1000)], 24, 1, 64, 8, None, 1, BF),   # more heads than a tile's rows
    "tokens_dim96": ([(1, 77), (1, 300)], 3, 3, 96, 24, None, 1, BF),
    "tokens_dim32": ([(1, 77), (1, 300)], 6, 3, 32, 1, 40, 1, FP),
    "waits": ([(1, 40), (0, 55), (1, 9), (0, 0)], 4, 4, 64, 16, None, 1, BF),
    "drafts": ([(5, 700), (3, 64), (1, 1), (4, 4)], 8, 2, 64, 16, None, 1, BF),
    "drafts_window": ([(5, 700), (3, 64), (1, 1), (4, 4)], 6, 2, 64, 16, 7, 3, FP),
    "chunk": ([(70, 70), (33, 300), (0, 12), (1, 64)], 4, 2, 64, 16, None, 1, BF),
    "chunk_dim128": ([(129, 200), (100, 1000)], 8, 2, 128, 32, None, 1, BF),
    "chunk_window": ([(150, 150), (97, 400)], 4, 1, 64, 16, 31, 1, BF),
    "chunk_dilated": ([(150, 150), (97, 400), (2, 3)], 4, 2, 32, 5, 9, 7, FP),
    "chunk_fp32": ([(57, 57), (31, 200)], 4, 2, 32, 16, 63, 2, F32),
    "chunk_kernel1": ([(20, 60)], 2, 2, 64, 16, 1, 1, BF),
    "kernel_past_all": ([(20, 60)], 2, 2, 64, 16, 2 ** 31 - 1, 1, BF),
    "dilation_past_all": ([(20, 60)], 2, 2, 64, 16, 3, 2 ** 31 - 1, BF),
    "odd_dim": ([(9, 100), (1, 40)], 3, 1, 20, 16, None, 1, BF),
    "odd_dim_window": ([(9, 100), (1, 40)], 3, 1, 17, 16, 12, 2, F32),
    "dim256": ([(3, 300)], 2, 1, 256, 16, None, 1, BF),
    "long": ([(1, 20000), (1, 100)], 8, 1, 64, 64, None, 1, BF),
    "long_drafts_fp32": ([(2, 5000)], 2, 1, 32, 16, None, 1, F32),
    "many_sequences": ([(1, 1 + (37 * i) % 90) for i in range(300)], 2, 1, 64, 16, None, 1, BF),
    "chunk_fp32_dim128": ([(130, 200), (7, 300)], 6, 2, 128, 24, None, 1, F32),
    "chunk_fp32_dim96": ([(41, 90), (7, 30)], 4, 2, 96, 16, 25, 1, F32),
    "drafts_fp32": ([(5, 700), (3, 64), (1, 1), (4, 4)], 8, 2, 64, 16, None, 1, F32),
    "token_fp32_dim96": ([(1, 300), (1, 17)], 3, 3, 96, 8, 50, 3, F32),
    "chunk_wide": ([(70 - i % 7, 75 + (13 * i) % 90) for i in range(64)], 8, 8, 64, 16, None, 1, BF),
    "chunk_wide_window": ([(70 - i % 7, 75 + (13 * i) % 90) for i in range(64)], 8, 8, 32, 8, 21, 1, FP),
    "chunk_long": ([(70, 5000), (64, 2500), (3, 9)], 4, 2, 64, 16, None, 1, BF),
    "chunk_long_dim128": ([(70, 5000), (64, 2500)], 4, 2, 128, 64, 4500, 1, FP),
    "ragged_many": ([(1, 9000)] + [(1, 1 + (37 * i) % 90) for i in range(299)], 2, 1, 64, 64, None, 1, BF),
    "odd_dim_long": ([(2, 3000), (1, 700)], 2, 1, 20, 16, None, 1, BF),
    "long_drafts_dilated": ([(20, 9000), (17, 40)], 4, 2, 32, 16, 4000, 2, BF),
    "long_fp32_rows": ([(20, 3000), (9, 100)], 4, 2, 64, 16, None, 1, F32),
    "many_heads_rep3": ([(11, 260)], 9, 3, 128, 16, None, 1, FP),
}


@pytest.mark.parametrize("name", CASES)
def test_against_float64(name):
    rows, hq, hkv, dim, page, kernel, dil, dtype = CASES[name]
    p = Problem(rows, hq, hkv, dim, page, dtype, seed=len(name))
    check(p.run(kernel, dil), p, kernel, dil, what=name)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_value_dim_differs(dtype):
    p = Problem([(4, 90), (1, 33)], 4, 2, 64, 16, dtype, dim_v=40)
    check(p.run(), p)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_scales(scale, dtype):
    p = Problem([(4, 90), (1, 33), (40, 70)], 4, 2, 64, 16, dtype)
    check(p.run(scale=scale), p, scale=scale)


@pytest.mark.parametrize("tokens", [1, 6, 140])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_padding_is_cleared(tokens, dtype):
    """Every token past new_lens has zeros and -inf, at any padded length."""
    p = Problem([(min(1, tokens), 40), (0, 30), (tokens, tokens + 9)], 4, 2, 64, 16, dtype, tokens=tokens)
    check(p.run(), p)


def test_lengths_out_of_range():
    """More new tokens than the tensor holds, than the sequence has, negative
    counts, positions past the table: clamped, empty, or without keys there."""
    p = Problem([(3, 40), (3, 40), (3, 40), (3, 40), (3, 40)], 4, 2, 64, 16, BF)
    p.news = torch.tensor([7, -1, 3, 3, 3], dtype=torch.int32, device=DEV)
    p.lens = torch.tensor([40, 40, 2, -5, 90], dtype=torch.int32, device=DEV)
    check(p.run(), p)
    check(p.run(4, 1), p, 4, 1)
    check(p.run(4, 3), p, 4, 3)


def test_without_new_lens():
    p = Problem([(3, 40), (3, 3)], 4, 2, 64, 16, BF)
    out = na.na1d_paged(p.q, p.kp, p.vp, p.table, p.lens)
    assert torch.equal(out, p.run()[0])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 5, 80])
def test_absent_pages(new, dtype):
    """Entries that name no page, in the middle of the keys and at their
    ends, leave their keys out; rows with none left are empty."""
    p = Problem([(new, 300), (new, 200), (new, 90)], 4, 2, 64, 16, dtype)
    for b, i, v in ((0, 3, -1), (0, 4, 2 ** 31 - 1), (0, 18, p.kp.shape[0]), (1, 0, -2 ** 31), (1, 12, -7)):
        p.table[b, i] = v
    p.table[2] = -1
    check(p.run(), p)
    check(p.run(40, 2), p, 40, 2)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new, kernel, dil", [(1, 20, 1), (6, 20, 1), (6, 5, 3), (90, 20, 1), (90, 7, 2), (90, None, 1)])
def test_nonfinite_outside_the_window(new, kernel, dil, dtype):
    """Keys and values that a query does not attend to may hold anything:
    behind its window, after it, in unused slots and pages."""
    p = Problem([(new, 200), (new, 131)], 4, 2, 64, 16, dtype, spare=3)
    want = p.run(kernel, dil)
    used = torch.zeros(p.kp.shape[:2], dtype=torch.bool)
    for b, (n, length) in enumerate(p.rows):
        for j in range(length):
            reach = any(pos >= j and (kernel is None or ((pos - j) % dil == 0 and pos - j < kernel * dil))
                        for pos in range(length - n, length))
            if reach:
                used[p.table[b, j // 16], j % 16] = True
    for bad in (math.nan, math.inf, -math.inf):
        for t in (p.kp, p.vp):
            t[~used.to(DEV)] = bad
        got = p.run(kernel, dil)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_nonfinite_in_cut_and_wide_calls(dtype):
    """As above where keys are cut into parts (few rows and many) and on tall
    tiles of many sequences: unused slots and keys behind every window."""
    for rows, hq, hkv, kernel in (([(5, 6000)], 4, 2, 3000), ([(70, 6000)], 4, 2, 3000), ([(2, 6000)], 4, 2, None),
                                  ([(70, 110)] * 64, 8, 8, 20)):
        p = Problem(rows, hq, hkv, 64, 16, dtype, spare=3)
        want = p.run(kernel)
        new, length = rows[0]
        first = 0 if kernel is None else max(0, length - new - kernel + 1)
        used = torch.zeros(p.kp.shape[:2], dtype=torch.bool, device=DEV)
        for b in range(len(rows)):
            keys = torch.arange(first, length, device=DEV)
            used[p.table[b, keys // 16].long(), keys % 16] = True
        for bad in (math.nan, math.inf):
            p.kp[~used] = bad
            p.vp[~used] = bad
            # within the used ones: the first key, seen by the first new token only
            if kernel is not None:
                for b in range(len(rows)):
                    p.vp[p.table[b, first // 16].long(), first % 16] = bad
            got = p.run(kernel)
            rest = slice(0, None) if kernel is None else slice(1, None)
            assert torch.isfinite(got[0][:, rest]).all()
            if kernel is None:
                assert torch.equal(got[0], want[0])
            else:
                # rows of a redone tile sum in another order: each of the two
                # is within the module's bound of the exact value, whose
                # magnitudes are at most max |v| and the product of norms
                norms = p.q.float().norm(dim=-1).max() * p.kp[used].float().norm(dim=-1).max() * 64 ** -0.5
                v = p.vp[used].float()
                top = v[torch.isfinite(v)].abs().max()
                step = torch.finfo(dtype).eps / 2
                rel = (8 + length ** 0.5 + 2 * (64 + 4) * norms) * 2.0 ** -24 + (step if dtype == BF else 0) + step
                assert ((got[0] - want[0])[:, rest].float().abs() <= 2 * rel * top).all()
            assert torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new, kernel, dil", [(6, 3, 1), (40, 5, 2), (90, 20, 1)])
def test_nonfinite_value_reaches_its_own_queries_only(new, kernel, dil, dtype):
    """A value of one of the new tokens is infinite: the queries whose
    windows hold it get it, in that dim, the others nothing."""
    p = Problem([(new, 200)], 4, 2, 64, 16, dtype)
    at = 200 - new + new // 2
    clean = p.run(kernel, dil)[0]
    p.vp[p.table[0, at // 16].long(), at % 16, 1, 37] = math.inf
    out = p.run(kernel, dil)[0]
    hit = torch.zeros_like(out, dtype=torch.bool)
    for i in range(new):
        back = 200 - new + i - at
        if back >= 0 and back % dil == 0 and back < kernel * dil:
            hit[0, i, 2:, 37] = True
    assert (out[hit] == math.inf).all()
    tol = 0.0 if dtype == F32 else 2 * torch.finfo(dtype).eps  # rows of a redone tile round their sums elsewhere
    diff = (out[~hit].float() - clean[~hit].float()).abs()
    assert (diff <= tol * clean[~hit].float().abs().clamp(min=0.25) + 1e-6).all()


def test_strides_and_orders():
    """Pages with heads outside of slots, padded rows, tables and queries as
    views: the results of the plain layout, bit for bit."""
    for dtype, new in ((BF, 1), (BF, 50), (F32, 3)):
        p = Problem([(new, 300), (new, 77)], 4, 2, 64, 16, dtype)
        want = p.run(50, 1)
        kp, vp, q, table = p.kp, p.vp, p.q, p.table
        p.kp = kp.transpose(1, 2).contiguous().transpose(1, 2)
        p.vp = torch.cat((vp, vp), -1)[..., :64]
        p.q = torch.cat((q, q), 2)[:, :, :4]
        p.table = torch.cat((table, table), 1)[:, :table.shape[1]]
        got = p.run(50, 1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        p.table = table.t().contiguous().t()
        got = p.run(50, 1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # single elements at odd offsets: other kernels, the same values within bounds
        p.kp = torch.cat((kp, kp), -1)[..., 1:65]
        p.table = table.long()
        p.lens, p.news = p.lens.long(), p.news.long()
        check(p.run(50, 1), p, 50, 1)


def test_shared_pages():
    """Two sequences that share the pages of a common prefix."""
    p = Problem([(1, 100), (1, 90)], 4, 2, 64, 16, BF)
    p.table[1, :3] = p.table[0, :3]
    check(p.run(), p)


def test_offsets_past_31_bits():
    """A pool whose last pages lie past 2^32 bytes and 2^31 elements."""
    pages, page, hkv, dim = 140000, 64, 2, 128
    kp = torch.zeros(pages, page, hkv, dim, dtype=BF, device=DEV)
    p = Problem([(1, 300), (40, 200)], 4, 2, 128, 64, BF)
    at = torch.arange(p.kp.shape[0]) * 11 + (pages - 11 * p.kp.shape[0])
    big_k, big_v = kp, torch.zeros_like(kp)
    big_k[at.to(DEV)], big_v[at.to(DEV)] = p.kp, p.vp
    want = p.run()
    table = torch.where(p.table >= 0, at.to(DEV, torch.int32)[p.table.long().clamp(min=0)], -1).to(torch.int32)
    assert big_k.numel() > 2 ** 31
    got = na.na1d_paged(p.q, big_k, big_v, table, p.lens, new_lens=p.news, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    k, v = _randn(1, 2, 40, 2, 128, dtype=BF), _randn(2, 2, 40, 2, 128, dtype=BF)
    na.na1d_paged_append(k, v, big_k, big_v, table, p.lens, p.news)
    na.na1d_paged_append(k, v, p.kp, p.vp, p.table, p.lens, p.news)
    assert torch.equal(big_k[at.to(DEV)], p.kp) and torch.equal(big_v[at.to(DEV)], p.vp)


def test_two_runs_agree():
    """Split keys are joined in a fixed order: the same bits each time."""
    p = Problem([(1, 9000), (3, 4000), (2, 17)], 8, 2, 128, 16, BF)
    first = p.run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(p.run(), first))


def test_refusals_on_the_device():
    p = Problem([(1, 40)], 4, 2, 64, 16, BF)
    with pytest.raises(RuntimeError, match="same GPU|must live on"):
        na.na1d_paged(p.q, p.kp, p.vp, p.table.cpu(), p.lens)
    with pytest.raises(TypeError, match="mixed dtypes"):
        na.na1d_paged(p.q.half(), p.kp, p.vp, p.table, p.lens)
    with pytest.raises(TypeError, match="float32"):
        na.na1d_paged(p.q.double(), p.kp.double(), p.vp.double(), p.table, p.lens)
    big = torch.zeros(1, 1, 1, 264, device=DEV)
    with pytest.raises(NotImplementedError, match="above 256"):
        na.na1d_paged(big, big, big, p.table, p.lens)


def test_no_tokens():
    p = Problem([(1, 40)], 4, 2, 64, 16, BF)
    out, lse = na.na1d_paged(p.q[:, :0], p.kp, p.vp, p.table, p.lens, return_lse=True)
    assert out.shape == (1, 0, 4, 64) and lse.shape == (1, 0, 4)
    kp = p.kp.clone()
    na.na1d_paged_append(p.q[:, :0, :2], p.q[:, :0, :2], p.kp, p.vp, p.table, p.lens)
    assert torch.equal(kp, p.kp)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

# rows (new, length), heads q/kv, dim, dim_v, page, plan, dtype
APPENDS = {
    "token": ([(1, 1), (1, 17), (0, 30), (1, 300)], 8, 2, 64, 64, 16, dict(dim=64), BF),
    "prompt": ([(70, 70), (33, 90), (0, 5)], 4, 4, 128, 128, 32, dict(dim=128, interleaved=True), FP),
    "part": ([(9, 40), (3, 3)], 3, 1, 80, 80, 5, dict(dim=20, scaling="linear", factor=4), BF),
    "odd": ([(9, 40), (3, 3)], 3, 1, 7, 5, 1, dict(dim=6, interleaved=True), F32),
    "plain": ([(4, 100), (2, 33)], 4, 2, 64, 64, 16, None, BF),
    "ramp": ([(5, 100005)], 2, 2, 32, 32, 64, dict(dim=32, scaling="ramp", factor=8, original_length=4096), F32),
}


@pytest.mark.parametrize("with_query", [True, False])
@pytest.mark.parametrize("name", APPENDS)
def test_append(name, with_query):
    rows, hq, hkv, dim, dim_v, page, plan, dtype = APPENDS[name]
    p = Problem(rows, hq, hkv, dim, page, dtype, dim_v=dim_v)
    plan = None if plan is None else na.RotaryPlan(**plan)
    B, L = p.q.shape[:2]
    k, v = _randn(11, B, L, hkv, dim, dtype=dtype), _randn(12, B, L, hkv, dim_v, dtype=dtype)
    kp, vp = p.kp.clone(), p.vp.clone()
    out = na.na1d_paged_append(k, v, p.kp, p.vp, p.table, p.lens, p.news, query=p.q if with_query else None, plan=plan)
    assert (out is None) == (not with_query)
    written = torch.zeros(kp.shape[:2], dtype=torch.bool, device=DEV)
    for b, (n, length) in enumerate(rows):
        if with_query:
            assert (out[b, n:] == 0).all()
        if n == 0:
            continue
        pos = torch.arange(length - n, length, device=DEV)
        pg, slot = p.table[b, pos // page].long(), pos % page
        written[pg, slot] = True
        assert torch.equal(p.vp[pg, slot], v[b, :n])
        if plan is None:
            assert torch.equal(p.kp[pg, slot], k[b, :n])
            assert not with_query or torch.equal(out[b, :n], p.q[b, :n])
            continue
        # the turn of rotary at these positions, bit for bit, and the formula
        turned = na.rotary(k[b:b + 1, :n], plan, pos)
        assert torch.equal(p.kp[pg, slot], turned[0])
        check_turn(turned, k[b:b + 1, :n], plan, pos)
        if with_query:
            assert torch.equal(out[b:b + 1, :n], na.rotary(p.q[b:b + 1, :n], plan, pos))
    assert torch.equal(p.kp[~written], kp[~written]) and torch.equal(p.vp[~written], vp[~written])


def test_append_to_absent_pages_and_bad_lengths():
    """Tokens without a page, before position 0 or past the table are not
    written; their queries are turned where they have a position."""
    p = Problem([(3, 40)] * 6, 4, 2, 64, 16, BF)
    p.table[0, 2] = -1
    p.table[1, 2] = p.kp.shape[0]
    p.lens = torch.tensor([40, 40, 2, -4, 49, 40], dtype=torch.int32, device=DEV)
    p.news = torch.tensor([3, 3, 3, 3, 3, -2], dtype=torch.int32, device=DEV)
    plan = na.RotaryPlan(64)
    k, v = _randn(1, 6, 3, 2, 64, dtype=BF), _randn(2, 6, 3, 2, 64, dtype=BF)
    kp, vp = p.kp.clone(), p.vp.clone()
    out = na.na1d_paged_append(k, v, p.kp, p.vp, p.table, p.lens, p.news, query=p.q, plan=plan)
    want = vp.clone()
    for b, i, pos in ((2, 1, 0), (2, 2, 1), (4, 0, 46), (4, 1, 47)):
        want[p.table[b, pos // 16].long(), pos % 16] = v[b, i]
    assert torch.equal(p.vp, want)
    assert torch.equal((p.kp != kp).any(-1).any(-1), (want != vp).any(-1).any(-1))
    assert (out[2, 0] == 0).all() and (out[3] == 0).all() and (out[5] == 0).all()
    for b, lo in ((0, 37), (1, 37), (4, 46)):
        assert torch.equal(out[b:b + 1], na.rotary(p.q[b:b + 1], plan, torch.arange(lo, lo + 3, device=DEV)))


def test_append_strides():
    p = Problem([(5, 40), (2, 20)], 4, 2, 64, 16, BF)
    plan = na.RotaryPlan(32)
    qkv = _randn(1, 2, 5, 8, 64, dtype=BF)
    q, k, v = qkv.split((4, 2, 2), 2)
    want_k, want_v = p.kp.clone(), p.vp.clone()
    want = na.na1d_paged_append(k.contiguous(), v.contiguous(), want_k, want_v, p.table, p.lens, p.news,
                                query=q.contiguous(), plan=plan)
    kp = p.kp.transpose(1, 2).contiguous().transpose(1, 2)
    vp = torch.cat((p.vp, p.vp), -1)[..., 3:67].clone()
    vp = torch.cat((p.vp, p.vp), -1)
    got = na.na1d_paged_append(k, v, kp, vp[..., :64], p.table.long(), p.lens.long(), p.news.long(), query=q, plan=plan)
    assert torch.equal(got, want) and torch.equal(kp, want_k) and torch.equal(vp[..., :64], want_v)
    assert torch.equal(vp[..., 64:], p.vp)
    odd = torch.cat((p.kp, p.kp), -1)[..., 1:65]
    odd.copy_(p.kp)
    na.na1d_paged_append(k, v, odd, vp[..., :64], p.table, p.lens, p.news, plan=plan)
    assert torch.equal(odd, want_k)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype, dilation", [(F32, 1), (F32, 3), (BF, 1), (BF, 4)])
def test_serving_follows_na1d(dtype, dilation):
    """A prompt in two chunks, then tokens one by one, through rotary, append
    and attention: the rows of na1d over the whole sequence."""
    torch.manual_seed(3)
    length, hq, hkv, dim, kernel = 61, 4, 2, 32, 9
    plan = na.RotaryPlan(32, scaling="linear", factor=2)
    q, k, v = (_randn(i, 2, length, h, dim, dtype=dtype) for i, h in enumerate((hq, hkv, hkv)))
    tq, tk = na.rotary_qk(q, k, plan)
    want = na.na1d(tq, tk, v, kernel_size=kernel, dilation=dilation, is_causal=True)
    cache = na.PagedKVCache(32, 4, 2, hkv, dim, dtype=dtype, device=DEV)
    layer = cache.layer(0)
    got, at = [], 0
    for n in (30, 25, 1, 1, 1, 3):
        part = slice(at, at + n)
        cache.reserve(n)
        turned = layer.append(k[:, part], v[:, part], query=q[:, part], plan=plan)
        got.append(layer.attend(turned, kernel, dilation))
        cache.trim(kernel, dilation)
        at += n
    got = torch.cat(got, 1)
    assert cache.free_pages > 0
    tol = 1e-5 if dtype == F32 else 4 * torch.finfo(dtype).eps
    assert torch.allclose(got.float(), want.float(), atol=tol, rtol=tol)


@pytest.mark.parametrize("gqa", [False, True])
def test_module_with_cache(gqa):
    """A stack of two causal modules answers token by token what it gives for
    the whole sequence; requests wait, end and start anew."""
    torch.manual_seed(1)
    dim, heads, kernel = 64, 4, 5
    layers = [na.NeighborhoodAttention1D(dim, heads, kernel, dilation=2, is_causal=True,
                                         num_kv_heads=2 if gqa else None, rotary=na.RotaryPlan(16)).to(DEV)
              for _ in range(2)]
    x = _randn(5, 2, 24, dim)

    def whole(y):
        for m in layers:
            y = y + m(y)
        return y

    cache = na.PagedKVCache(24, 4, 2, 2 if gqa else heads, 16, layers=2, dtype=torch.float32, device=DEV)

    def step(y, counts):
        cache.reserve(counts)
        for i, m in enumerate(layers):
            y = y + m(y, cache=cache.layer(i))
        cache.trim(kernel, 2)
        return y

    with torch.no_grad():
        want = whole(x)
        first = step(torch.cat((x[:, :10], x.new_full((2, 2, dim), 9.0)), 1), [10, 7])
        assert torch.allclose(first[0, :10], want[0, :10], atol=1e-5)
        assert torch.allclose(first[1, :7], want[1, :7], atol=1e-5)
        second = step(torch.stack((x[0, 10:11], x[1, 7:8])), [1, 0])
        assert torch.allclose(second[0], want[0, 10:11], atol=1e-5)
        for i in range(11, 24):
            y = step(torch.stack((x[0, i:i + 1], x[1, i - 4:i - 3])), 1)
            assert torch.allclose(y[0], want[0, i:i + 1], atol=1e-5)
            assert torch.allclose(y[1], want[1, i - 4:i - 3], atol=1e-5)
        cache.release(1)
        again = step(x[:, :5].flip(0), [0, 5])
        assert torch.allclose(again[1], want[0, :5], atol=1e-5)
        with torch.enable_grad(), pytest.raises(RuntimeError, match="no gradients"):
            layers[0](x[:, :5], cache=cache.layer(0))


def test_merge_with_other_keys():
    """lse joins the cache with other keys: half of the keys each."""
    p = Problem([(3, 100), (3, 60)], 4, 2, 64, 16, F32)
    whole, lse = p.run()
    left, right = p.table.clone(), p.table.clone()
    left[:, 2:], right[:, :2] = -1, -1
    p.table = left
    a = p.run()
    p.table = right
    b = p.run()
    out, l = na.merge_attentions([a[0], b[0]], [a[1], b[1]])
    assert torch.allclose(out, whole, atol=2e-6) and torch.allclose(l, lse, atol=2e-6)


def test_another_stream():
    p = Problem([(1, 4000), (2, 500)], 8, 2, 64, 16, BF)
    want = p.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = p.run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_steps_follow_the_cache():
    """Two captured steps (with cut keys, so with a workspace each) replayed
    as lengths grow, eager work between the replays."""
    cache = na.PagedKVCache(300, 16, 2, 2, 64, device=DEV)
    layer = cache.layer(0)
    plan = na.RotaryPlan(64)
    plan.table(DEV)
    cache.reserve([2000, 900])
    k, v = _randn(1, 2, 2000, 2, 64, dtype=BF), _randn(2, 2, 2000, 2, 64, dtype=BF)
    layer.append(k, v, plan=plan)
    cache.reserve(1)
    q1, k1, v1 = (_randn(3 + i, 2, 1, h, 64, dtype=BF) for i, h in enumerate((8, 2, 2)))

    def step():
        turned = layer.append(k1, v1, query=q1, plan=plan)
        return layer.attend(turned, return_lse=True), layer.attend(turned, 700, return_lse=True)

    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for i in range(4):
        if i:
            cache.reserve([1, i])
        for t in (q1, k1, v1):
            t.copy_(_randn(20 + i, *t.shape, dtype=BF))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for got in outs:
            for a, b in zip(got, want):
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_without_the_host_binding(dtype, monkeypatch):
    """The ctypes calls give what the C++ host binding gives."""
    from natten_mps_amd._core import _lib

    plan = na.RotaryPlan(32, scaling="linear", factor=4)
    p = Problem([(3, 700), (40, 90)], 4, 2, 64, 16, dtype)
    k, v = _randn(1, 2, 40, 2, 64, dtype=dtype), _randn(2, 2, 40, 2, 64, dtype=dtype)
    pos = torch.arange(80, device=DEV).view(2, 40)
    leaf, g = _randn(3, 2, 40, 2, 64, dtype=dtype).requires_grad_(), _randn(4, 2, 40, 2, 64, dtype=dtype)

    def calls():
        kp, vp = p.kp.clone(), p.vp.clone()
        q = na.na1d_paged_append(k, v, kp, vp, p.table, p.lens, p.news, query=p.q, plan=plan)
        plain = na.na1d_paged_append(k, v, kp, vp, p.table, p.lens, p.news, query=p.q)
        att = na.na1d_paged(q, kp, vp, p.table, p.lens, 300, 2, new_lens=p.news, return_lse=True)
        every = na.na1d_paged(q, kp, vp, p.table, p.lens, new_lens=p.news)
        out = na.rotary(leaf, plan, pos)
        both = na.rotary_qk(leaf, g, plan)
        return (q, plain, kp, vp, *att, every, out, *both, *torch.autograd.grad(out, leaf, g),
                *torch.autograd.grad(both[0], leaf, g))

    with_binding = calls()
    monkeypatch.setattr(_lib, "binding", lambda: None)
    for a, b in zip(with_binding, calls()):
        assert torch.equal(a, b)
