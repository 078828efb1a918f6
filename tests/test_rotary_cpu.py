"""Rotary plans and the paged cache's bookkeeping without a GPU: frequencies
against the formulas, fixed-point turns against exact rationals, refusals of
every entry point, and pages handed out, given back and trimmed."""
from __future__ import annotations

import copy
import ctypes
import math
import pickle
from fractions import Fraction

import pytest
import torch

import natten_mps_amd as na
from natten_mps_amd._core import _lib


def _plan(**kw):
    return na.RotaryPlan(8, **kw)


def test_frequencies():
    f = [10000.0 ** (-2 * j / 8) for j in range(4)]
    assert _plan().frequencies == pytest.approx(f, rel=1e-15)
    assert _plan(base=500.0).frequencies == pytest.approx([500.0 ** (-2 * j / 8) for j in range(4)], rel=1e-15)
    assert _plan(scaling="linear", factor=4).frequencies == pytest.approx([x / 4 for x in f], rel=1e-15)
    based = _plan(scaling="base", factor=4).frequencies
    assert based[0] == 1.0 and based[-1] == pytest.approx(f[-1] / 4, rel=1e-14)
    # two axes of four dims each: two pairs an axis
    assert na.RotaryPlan(8, axes=2).frequencies == pytest.approx([1.0, 0.01], rel=1e-15)
    assert na.RotaryPlan(2, scaling="base", factor=4).frequencies == (1.0,)


def test_ramp():
    p = _plan(scaling="ramp", factor=8, original_length=4096, low=1, high=32)
    f = [10000.0 ** (-2 * j / 8) for j in range(4)]
    turns = [4096 * x / (2 * math.pi) for x in f]
    assert turns[0] > 32 and turns[1] > 32 and 1 < turns[2] < 32 and turns[3] < 1
    keep = (turns[2] - 1) / 31
    assert p.frequencies == pytest.approx([f[0], f[1], f[2] * (keep + (1 - keep) / 8), f[3] / 8], rel=1e-14)
    assert p.magnitude == pytest.approx(1 + 0.1 * math.log(8))
    assert _plan(scaling="ramp", factor=8, original_length=4096, magnitude=1.0).magnitude == 1.0


def test_turns_hold_the_frequency_modulo_a_turn():
    freqs = [1.0, -0.25, 7.0, 1e-9, 0.0, 2 * math.pi, 100.0, 3.0]
    p = na.RotaryPlan(16, frequencies=freqs)
    for f, t in zip(freqs, p._turns):
        assert -2 ** 63 <= t < 2 ** 63
        got = Fraction(t % 2 ** 64, 2 ** 64)
        want = Fraction(f) / (2 * Fraction(math.pi))  # the double's own value: 2 pi to 2^-53
        gap = (got - want) % 1
        # two roundings of f / 2 pi in double precision, absolute in turns
        assert min(gap, 1 - gap) <= Fraction(1, 2 ** 52) * (1 + abs(want))


def test_plan_is_a_value():
    p = na.RotaryPlan(12, axes=3, interleaved=True, scaling="linear", factor=2)
    assert p == na.RotaryPlan(12, axes=3, interleaved=True, scaling="linear", factor=2)
    assert hash(p) == hash(pickle.loads(pickle.dumps(p))) and pickle.loads(pickle.dumps(p)) == p
    assert copy.deepcopy(p) is p
    assert p != na.RotaryPlan(12, axes=3, scaling="linear", factor=2)
    with pytest.raises(AttributeError):
        p.dim = 4
    assert torch.equal(p.table("cpu"), torch.tensor(p._turns))


@pytest.mark.parametrize("kw, text", [
    (dict(dim=0), "multiple"), (dict(dim=3), "multiple"), (dict(dim=True), "multiple"),
    (dict(dim=8, axes=3), "multiple"), (dict(dim=8, axes=4), "axes"), (dict(dim=8, axes=True), "axes"),
    (dict(dim=8, scaling="other"), "scaling"), (dict(dim=8, factor=0.0), "factor"),
    (dict(dim=8, factor=math.nan), "factor"), (dict(dim=8, base=-1.0), "base"), (dict(dim=8, base=math.inf), "base"),
    (dict(dim=8, scaling="ramp", factor=2), "original_length"),
    (dict(dim=8, scaling="ramp", factor=2, original_length=0), "original_length"),
    (dict(dim=8, scaling="ramp", factor=2, original_length=8, low=4, high=4), "below"),
    (dict(dim=8, frequencies=[1.0]), "frequencies"), (dict(dim=8, frequencies=[1.0, 1.0, 1.0, math.inf]), "finite"),
    (dict(dim=8, frequencies=[1.0] * 4, scaling="linear"), "combined"), (dict(dim=8, magnitude="1"), "magnitude"),
])
def test_plan_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        na.RotaryPlan(kw.pop("dim"), **kw)


def test_rotary_refusals():
    x = torch.zeros(2, 5, 3, 8)
    p = _plan()
    with pytest.raises(ValueError, match="shape"):
        na.rotary(x[0], p)
    with pytest.raises(TypeError, match="RotaryPlan"):
        na.rotary(x, 8)
    with pytest.raises(ValueError, match="turns 8 dims"):
        na.rotary(x[..., :4], p)
    with pytest.raises(ValueError, match="explicit positions"):
        na.rotary(x[:, None], p)
    for bad in (torch.zeros(4, dtype=torch.int64), torch.zeros(3, 5, dtype=torch.int64),
                torch.zeros(2, 5, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="positions must have shape"):
            na.rotary(x, p, bad)
    with pytest.raises(ValueError, match="int32 or int64"):
        na.rotary(x, p, torch.zeros(5))
    with pytest.raises(ValueError, match="but for their heads"):
        na.rotary_qk(x, x[:, :4], p)
    with pytest.raises(ValueError, match="rotary plan has"):
        na.NeighborhoodAttention2D(16, 2, 3, rotary=p)
    with pytest.raises(ValueError, match="turns 8 dims"):
        na.NeighborhoodAttention1D(8, 2, 3, rotary=p)


def _cache_args(batch=2, tokens=3, hkv=2, dim=8, pages=4, page=5, width=3):
    return dict(key=torch.zeros(batch, tokens, hkv, dim), value=torch.zeros(batch, tokens, hkv, dim),
                key_pages=torch.zeros(pages, page, hkv, dim), value_pages=torch.zeros(pages, page, hkv, dim),
                block_table=torch.zeros(batch, width, dtype=torch.int32),
                seq_lens=torch.zeros(batch, dtype=torch.int32))


@pytest.mark.parametrize("over, text", [
    (dict(key=torch.zeros(2, 3, 8)), "expects key and value"),
    (dict(value=torch.zeros(2, 4, 2, 8)), "expects key and value"),
    (dict(key_pages=torch.zeros(4, 5, 16)), "expects pages"),
    (dict(value_pages=torch.zeros(4, 6, 2, 8)), "must match but for"),
    (dict(key_pages=torch.zeros(0, 5, 2, 8), value_pages=torch.zeros(0, 5, 2, 8)), "at least one page"),
    (dict(key_pages=torch.zeros(4, 5, 8, 2).transpose(2, 3)), "contiguous in their head dim"),
    (dict(key_pages=torch.zeros(1, 5, 2, 8).expand(4, 5, 2, 8)), "expanded"),
    (dict(block_table=torch.zeros(3, 3, dtype=torch.int32)), "block_table"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), "block_table"),
    (dict(block_table=torch.zeros(2, 3)), "int32 or int64"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), "seq_lens"),
    (dict(seq_lens=torch.zeros(2)), "int32 or int64"),
    (dict(new_lens=torch.zeros(2, 1, dtype=torch.int32)), "new_lens"),
    (dict(key=torch.zeros(2, 3, 1, 8), value=torch.zeros(2, 3, 1, 8)), "heads and dims"),
    (dict(query=torch.zeros(2, 2, 4, 8)), "query must be"),
    (dict(plan=na.RotaryPlan(16)), "turns 16 dims"),
    (dict(plan=na.RotaryPlan(8, axes=2)), "one axis"),
])
def test_append_refusals(over, text):
    with pytest.raises(ValueError, match=text):
        na.na1d_paged_append(**{**_cache_args(), **over})


def test_append_refuses_gradients():
    a = _cache_args()
    with pytest.raises(RuntimeError, match="no gradients"):
        na.na1d_paged_append(**{**a, "key": a["key"].requires_grad_()})


@pytest.mark.parametrize("over, text", [
    (dict(query=torch.zeros(2, 3, 8)), "expects query"),
    (dict(query=torch.zeros(2, 3, 4, 16)), "Head dim"),
    (dict(query=torch.zeros(2, 3, 3, 8)), "divisible"),
    (dict(kernel_size=0), "> 0"), (dict(kernel_size=True), "not bools"), (dict(kernel_size=(3, 3)), "length 1"),
    (dict(kernel_size=3, dilation=0), "> 0"), (dict(kernel_size=3, dilation=True), "not bools"),
    (dict(dilation=2), "needs a kernel_size"),
    (dict(seq_lens=torch.zeros(2, 1, dtype=torch.int32)), "seq_lens"),
    (dict(block_table=torch.zeros(6, dtype=torch.int32)), "block_table"),
    (dict(value_pages=torch.zeros(4, 5, 2, 8, 1)), "expects pages"),
])
def test_paged_refusals(over, text):
    a = _cache_args()
    a = dict(query=torch.zeros(2, 3, 4, 8), **{n: a[n] for n in ("key_pages", "value_pages", "block_table",
                                                                 "seq_lens")})
    with pytest.raises(ValueError, match=text):
        na.na1d_paged(**{**a, **over})


def test_paged_refuses_gradients():
    a = _cache_args()
    q = torch.zeros(2, 3, 4, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradients"):
        na.na1d_paged(q, a["key_pages"], a["value_pages"], a["block_table"], a["seq_lens"])


def _paged(**over):
    p = _lib.Paged()
    for n, v in dict(batch=2, tokens=3, heads_q=4, heads_kv=2, dim_qk=8, dim_v=8, dtype=_lib.F32, pages=4,
                     page_size=5, table_width=3, table_stride=3, kernel=0, dilation=1, scale=0.5).items():
        setattr(p, n, over.pop(n, v))
    for n in ("key_stride", "value_stride"):
        getattr(p, n)[:] = over.pop(n, (80, 16, 8))
    assert not over
    return p


@pytest.mark.parametrize("over, code, text", [
    (dict(batch=0), 1, "batch"), (dict(heads_q=3), 1, "divisible"), (dict(heads_q=0), 1, "heads"),
    (dict(dim_qk=257), 2, "above 256"), (dict(dim_v=0), 1, "head dims"), (dict(dtype=3), 1, "dtype"),
    (dict(pages=0), 1, "pages"), (dict(page_size=0), 1, "page_size"), (dict(table_width=0), 1, "table_width"),
    (dict(table_stride=-1), 1, "stride"), (dict(key_stride=(-1, 1, 1)), 1, "stride"), (dict(kernel=-1), 1, "kernel"),
    (dict(dilation=0), 1, "dilation"), (dict(dilation=2), 1, "needs a kernel"),
    (dict(batch=2 ** 20, tokens=2 ** 20), 2, "2\\^27"), (dict(batch=2 ** 16, tokens=2 ** 12), 2, "2\\^27"),
    (dict(table_width=2 ** 20, page_size=2 ** 11), 2, "positions"),
])
def test_paged_codes(over, code, text):
    import re

    lib, lay, d = _lib.load(), ctypes.byref(_lib.Layout()), ctypes.c_void_p(16)
    p = _paged(**over)
    rc = lib.natten_hip_paged_forward(ctypes.byref(p), d, d, None, d, lay, d, d, d, lay, d, lay, None, 0, None)
    assert rc == code and re.search(text, lib.natten_hip_last_error().decode())
    assert lib.natten_hip_paged_workspace(ctypes.byref(p)) == -1


def test_paged_workspace_is_checked():
    lib, lay, d = _lib.load(), ctypes.byref(_lib.Layout()), ctypes.c_void_p(16)
    p = _paged(table_width=1000, page_size=64)
    need = lib.natten_hip_paged_workspace(ctypes.byref(p))
    assert need > 0
    for work, size in ((None, need), (d, need - 1), (ctypes.c_void_p(24), need)):
        rc = lib.natten_hip_paged_forward(ctypes.byref(p), d, d, None, d, lay, d, d, d, lay, d, lay, work, size, None)
        assert rc == 1 and "workspace" in lib.natten_hip_last_error().decode()
    # short runs of keys are never cut
    assert lib.natten_hip_paged_workspace(ctypes.byref(_paged())) == 0


def test_null_operands():
    lib, lay, d = _lib.load(), ctypes.byref(_lib.Layout()), ctypes.c_void_p(16)
    p = ctypes.byref(_paged())
    assert lib.natten_hip_paged_forward(p, None, d, None, d, lay, d, d, d, lay, d, lay, None, 0, None) == 1
    assert "NULL" in lib.natten_hip_last_error().decode()
    assert lib.natten_hip_paged_append(p, None, None, d, d, None, d, lay, d, lay, d, lay, None, None, d, d, None) == 1
    r = _lib.Rotary()
    r.batch = r.heads_q = r.axes = 1
    r.length[:] = [1, 1, 4]
    r.dim = r.turned = 8
    assert lib.natten_hip_rotary(ctypes.byref(r), None, None, d, lay, d, lay, None, None, None, None, None) == 1
    assert lib.natten_hip_rotary(ctypes.byref(r), d, None, None, None, None, None, None, None, None, None, None) == 1
    for name, value, text in (("turned", 6, None), ("turned", 7, "multiple"), ("turned", 10, "multiple"),
                              ("axes", 0, "axes"), ("position_bits", 8, "position_bits"), ("dim", 300, "256"),
                              ("dtype", 5, "dtype"), ("batch", 0, "batch"), ("heads_q", 0, "heads")):
        if text is None:
            continue
        old = getattr(r, name)
        setattr(r, name, value)
        assert lib.natten_hip_rotary(ctypes.byref(r), d, None, d, lay, d, lay, None, None, None, None, None) in (1, 2)
        assert text in lib.natten_hip_last_error().decode()
        setattr(r, name, old)


def test_struct_layouts(tmp_path):
    import os
    import subprocess

    from conftest import ROOT

    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "natten_hip.h"\nint main(void) {\n'
                   'printf("%zu %zu %zu %zu %zu %zu %zu\\n", sizeof(natten_rotary_t), offsetof(natten_rotary_t, '
                   'magnitude), offsetof(natten_rotary_t, position_stride), sizeof(natten_paged_t), '
                   'offsetof(natten_paged_t, table_stride), offsetof(natten_paged_t, value_stride), '
                   'offsetof(natten_paged_t, scale));\nreturn 0;\n}\n')
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    R, P = _lib.Rotary, _lib.Paged
    assert got == [ctypes.sizeof(R), R.magnitude.offset, R.position_stride.offset, ctypes.sizeof(P),
                   P.table_stride.offset, P.value_stride.offset, P.scale.offset]


# ---------------------------------------------------------------------------
# the cache's bookkeeping
# ---------------------------------------------------------------------------


def _cache(**kw):
    return na.PagedKVCache(**{**dict(num_pages=10, page_size=4, batch=3, num_kv_heads=2, head_dim=8, max_pages=6,
                                     device="cpu", dtype=torch.float32), **kw})


def _held(c):
    """Pages named by the table, each at most once, and as many as are not free."""
    pages = [p for row in c.block_table.tolist() for p in row if p >= 0]
    assert len(set(pages)) == len(pages) and all(0 <= p < c.num_pages for p in pages)
    assert len(pages) + c.free_pages == c.num_pages
    return pages


def test_cache_reserves_and_releases():
    c = _cache()
    c.reserve([5, 0, 4])
    assert c.lengths == [5, 0, 4] == c.seq_lens.tolist() and c.new_lens.tolist() == [5, 0, 4]
    assert len(_held(c)) == 3
    first = c.block_table.clone()
    c.reserve(1)
    assert c.lengths == [6, 1, 5] and c.new_lens.tolist() == [1, 1, 1] and len(_held(c)) == 5
    assert torch.equal(c.block_table[0], first[0])  # room was left on its second page
    c.release(0)
    assert c.lengths == [0, 1, 5] and c.seq_lens.tolist() == [0, 1, 5] and c.new_lens.tolist()[0] == 0
    assert c.block_table[0].tolist() == [-1] * 6 and len(_held(c)) == 3
    c.reserve([1, 0, 0])
    assert len(_held(c)) == 4


def test_cache_refuses_what_does_not_fit():
    c = _cache()
    c.reserve([8, 8, 8])
    state = (c.lengths, c.block_table.clone(), c.seq_lens.clone(), c.free_pages)
    with pytest.raises(RuntimeError, match="pages needed"):
        c.reserve([8, 8, 8])
    with pytest.raises(RuntimeError, match="at most 6"):
        _cache(num_pages=100).reserve([25, 0, 0])
    for bad in ([1, 1], [1, -1, 1], [1, True, 1], [1, 1.0, 1]):
        with pytest.raises(ValueError):
            c.reserve(bad)
    assert (c.lengths, c.free_pages) == (state[0], state[3])
    assert torch.equal(c.block_table, state[1]) and torch.equal(c.seq_lens, state[2])
    with pytest.raises(IndexError):
        c.release(3)
    with pytest.raises(IndexError):
        c.release(-1)
    with pytest.raises(IndexError):
        c.layer(1)
    with pytest.raises(ValueError, match="page_size"):
        _cache(page_size=0)


def test_cache_trims_behind_the_window():
    c = _cache(num_pages=20, max_pages=10)
    c.reserve([17, 3, 30])
    before = c.block_table.clone()
    c.trim(5, 2)  # the next token of sequence 0 (at 17) reaches back to 9, of sequence 2 to 22
    t = c.block_table
    assert t[0, :2].tolist() == [-1, -1] and torch.equal(t[0, 2:], before[0, 2:])
    assert torch.equal(t[1], before[1])
    assert t[2, :5].tolist() == [-1] * 5 and torch.equal(t[2, 5:], before[2, 5:])
    _held(c)
    c.reserve([4, 0, 0])
    assert c.lengths[0] == 21 and t[0, 5] >= 0
    c.release(2)
    c.release(0)
    c.release(1)
    assert c.free_pages == 20


def test_module_with_cache_refusals():
    layer = _cache().layer(0)
    x = torch.zeros(3, 1, 16)
    for kw in (dict(), dict(is_causal=True, stride=2), dict(is_causal=True, attn_drop=0.1)):
        with torch.no_grad(), pytest.raises(ValueError, match="a cache needs"):
            na.NeighborhoodAttention1D(16, 2, 3, **kw)(x, cache=layer)
    with pytest.raises(ValueError, match="exclude"):
        na.NeighborhoodAttention1D(16, 2, 3, is_causal=True)(x, torch.tensor([1, 1, 1]), cache=layer)
