"""Measured cases of rotary positions and of 1-D causal neighbourhood
attention over a paged cache: what a program that trains such layers, and one
that answers requests with them, has these operators do.

A case is a dict of plain values; a size is a text with one number per axis
("56x56").  ``op`` names the operator:

* ``rotary``: ``rotary_qk`` turns queries and keys ``[B, *size, heads, dim]``
  by the angles of their positions, with the gradients of both when ``grad``;
* ``append``: ``na1d_paged_append`` turns the keys of the new tokens by their
  positions and writes keys and values to the pages of a cache, and turns the
  queries on the way;
* ``paged``: ``na1d_paged``, the attention of ``new`` new tokens a sequence
  over the paged cache (``kernel`` 0: every key up to the token's own).

``own`` chooses between the package's kernels and the plain form below
(elementary torch operations in 32 bits, angles in 64); ``exact`` restates
the operators in float64.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DEV = "cuda"


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "natten-mps_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import natten_mps_amd

    return natten_mps_amd


_ROTARY = dict(op="rotary", dtype="bfloat16", batch=1, size="128", heads=4, kv_heads=4, dim=32, turned=32,
               interleaved=False, scaling="none", factor=1.0, start=0, packed=False, grad=True)
_APPEND = dict(op="append", dtype="bfloat16", batch=1, new=1, shortest_new=1, cached=1024, shortest_cached=1,
               heads=8, kv_heads=2, dim=64, turned=64, interleaved=False, scaling="none", factor=1.0, page=16)
_PAGED = dict(op="paged", dtype="bfloat16", batch=1, new=1, shortest_new=1, cached=1024, shortest_cached=1,
              heads=8, kv_heads=2, dim=64, kernel=0, dilation=1, page=16)


def _case(**over):
    return dict({"rotary": _ROTARY, "append": _APPEND, "paged": _PAGED}[over["op"]], **over)


def _ints(text):
    return tuple(int(x) for x in text.split("x"))


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # a short single-precision sequence layer, forward only: latency
        _case(name="rotary_line_fp32", op="rotary", dtype="float32", batch=2, size="128", grad=False),
        # a training step of a long-context layer with grouped heads, far
        # positions and frequencies stretched by parts
        _case(name="rotary_line_step", op="rotary", batch=4, size="16384", heads=8, kv_heads=2, dim=64, turned=64,
              scaling="ramp", factor=8.0, start=500000),
        # the first level of an image backbone: adjacent pairs, q and k as
        # views of the packed projection
        _case(name="rotary_plane_step", op="rotary", dtype="float16", batch=64, size="56x56", heads=4, kv_heads=4,
              dim=32, turned=32, interleaved=True, packed=True),
        # a video layer: three axes share 48 of 64 dims, the rest stays
        _case(name="rotary_volume_step", op="rotary", batch=2, size="16x32x32", heads=8, kv_heads=8, dim=64,
              turned=48),
        # one new token of each of 64 requests
        _case(name="append_token", op="append", batch=64, cached=16384, shortest_cached=1),
        # prompts of different lengths, padded to one batch
        _case(name="append_prompt", op="append", dtype="float16", batch=4, new=4096, shortest_new=1025, cached=0,
              shortest_cached=0, heads=32, kv_heads=8, dim=128, turned=128, interleaved=True, page=64),
        # one new token of a few requests, a narrow dilated window: the
        # smallest call of all
        _case(name="token_window", op="paged", batch=8, cached=4096, kernel=33, dilation=4),
        # one new token of each of 32 requests over all of their tokens: the
        # traffic of a serving step
        _case(name="token_ragged", op="paged", batch=32, cached=16384, shortest_cached=37, heads=32, kv_heads=8,
              dim=128),
        # a few drafted tokens of one request with a very long context
        _case(name="token_far", op="paged", dtype="float16", batch=1, new=5, shortest_new=5, cached=131065,
              shortest_cached=131065, heads=8, kv_heads=1, dim=64, page=64),
        # chunks of long prompts in a window of about a thousand keys
        _case(name="chunk_window", op="paged", batch=4, new=2048, shortest_new=517, cached=14000,
              shortest_cached=100, kernel=1025),
        # a chunk of a long prompt over everything before it, the largest call
        _case(name="chunk_full", op="paged", batch=2, new=4096, shortest_new=4001, cached=28000,
              shortest_cached=17003, heads=16, kv_heads=4, dim=128, page=32),
        # a short single-precision chunk of an odd length, dilated
        _case(name="chunk_fp32", op="paged", dtype="float32", batch=2, new=257, shortest_new=131, cached=1000,
              heads=4, kv_heads=4, dim=32, kernel=63, dilation=2),
    ]


# What a draw keeps under: elements that a rotary or append call moves,
# multiplications of an attention call and the elements of its cache.
_MOST_ELEMENTS = 64 << 20
_MOST_FLOPS = 1.6e12
_MOST_FLOPS_FP32 = 4e10
_MOST_CACHE = 512 << 20


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_turned(rng, dim, axes):
    """Dims that a rotation of `axes` axes takes of a head of `dim`."""
    unit = 2 * axes
    if rng.random() < 0.6:
        return dim // unit * unit
    return rng.randint(1, dim // unit) * unit


def draw(rng):
    while True:
        op = rng.choice(("rotary", "append", "paged", "paged"))
        c = {"rotary": _draw_rotary, "append": _draw_append, "paged": _draw_paged}[op](rng)
        if c is not None:
            return c


def _draw_heads(rng):
    kv = rng.choice((1, 2, 3, 4, 8))
    return kv * rng.choice((1, 1, 2, 3, 4, 8)), kv


def _draw_rotary(rng):
    rank = rng.choice((1, 1, 2, 3))
    if rank == 1:
        size = (_log_int(rng, 1, 65536),)
    elif rank == 2:
        size = tuple(_log_int(rng, 7, 256) for _ in range(2))
    else:
        size = (_log_int(rng, 2, 24),) + tuple(_log_int(rng, 7, 64) for _ in range(2))
    heads, kv_heads = _draw_heads(rng)
    packed = rng.random() < 0.3
    if packed:
        kv_heads = heads
    dim = rng.choice((16, 32, 48, 64, 80, 96, 128, 192))
    scaling = rng.choice(("none", "none", "linear", "base", "ramp"))
    per = math.prod(size) * (heads + kv_heads) * dim
    if per > _MOST_ELEMENTS:
        return None
    return _case(op="rotary", dtype=rng.choice(("bfloat16", "bfloat16", "float16", "float32")),
                 batch=_log_int(rng, 1, max(1, min(64, _MOST_ELEMENTS // per))), size="x".join(map(str, size)),
                 heads=heads, kv_heads=kv_heads, dim=dim, turned=_draw_turned(rng, dim, rank),
                 interleaved=rng.random() < 0.5, scaling=scaling,
                 factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0, 32.0)),
                 start=rng.choice((0, 1, 4095, 1000003)) if rank == 1 else 0, packed=packed,
                 grad=rng.random() < 0.6)


def _draw_append(rng):
    heads, kv_heads = _draw_heads(rng)
    dim = rng.choice((32, 64, 80, 96, 128))
    new = rng.choice((1, 1, _log_int(rng, 2, 16), _log_int(rng, 16, 8192)))
    cached = rng.choice((0, _log_int(rng, 1, 65536)))
    batch = _log_int(rng, 1, 256)
    if batch * new * (heads + 2 * kv_heads) * dim > _MOST_ELEMENTS:
        return None
    if batch * (cached + new) * kv_heads * dim > _MOST_CACHE // 8:
        return None
    scaling = rng.choice(("none", "none", "linear", "base", "ramp"))
    return _case(op="append", dtype=rng.choice(("bfloat16", "bfloat16", "float16", "float32")), batch=batch, new=new,
                 shortest_new=rng.randint(0, new) if new > 1 else new, cached=cached,
                 shortest_cached=rng.randint(0, cached), heads=heads, kv_heads=kv_heads, dim=dim,
                 turned=_draw_turned(rng, dim, 1), interleaved=rng.random() < 0.5, scaling=scaling,
                 factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0, 32.0)),
                 page=rng.choice((1, 8, 16, 16, 24, 32, 64, 128, 256)))


def _draw_paged(rng):
    heads, kv_heads = _draw_heads(rng)
    new = rng.choice((1, 1, 1, _log_int(rng, 2, 16), _log_int(rng, 16, 4096)))
    cached = rng.choice((0, _log_int(rng, 1, 131072), _log_int(rng, 64, 32768), _log_int(rng, 64, 32768)))
    kernel = rng.choice((0, 0, _log_int(rng, 1, 16), _log_int(rng, 16, 8192)))
    c = _case(op="paged", dtype=rng.choice(("bfloat16", "bfloat16", "float16", "float32")),
              batch=_log_int(rng, 1, 256), new=new, shortest_new=rng.randint(0, new) if new > 1 else new,
              cached=cached, shortest_cached=rng.randint(0, cached), heads=heads, kv_heads=kv_heads,
              dim=rng.choice((32, 64, 64, 96, 128, 128)), kernel=kernel,
              dilation=rng.choice((1, 1, 2, 4, 7)) if kernel else 1,
              page=rng.choice((1, 8, 16, 16, 24, 32, 64, 128, 256)))
    # a single-precision head of 128 dims or a row of every head and token
    # has to stay a case that the plain form does in a second
    if c["batch"] * (cached + new) * kv_heads * c["dim"] > _MOST_CACHE:
        return None
    if work(c)["flops"] > (_MOST_FLOPS_FP32 if c["dtype"] == "float32" else _MOST_FLOPS):
        return None
    return c


# ---------------------------------------------------------------------------
# lengths and frequencies
# ---------------------------------------------------------------------------


def _spread(lo, hi, n):
    """n lengths from hi down to lo, evenly; [hi] alone for n = 1."""
    return [hi - (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _lengths(case):
    """(new tokens, cached tokens) of each sequence, a fixed set per case:
    long prompts are not the ones with long caches."""
    new = _spread(case["shortest_new"], case["new"], case["batch"])
    cached = _spread(case["shortest_cached"], case["cached"], case["batch"])
    return list(zip(new, reversed(cached) if case["batch"] > 1 else cached))


_ORIGINAL_LENGTH = 4096
_LOW, _HIGH = 1.0, 32.0


def _frequencies(case, axes):
    """Angle per position of each pair of one axis (float64), and the factor
    on cosine and sine."""
    n, s = case["turned"] // axes, case["factor"]
    base, magnitude = 10000.0, 1.0
    if case["scaling"] == "base" and n > 2:
        base *= s ** (n / (n - 2))
    f = base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if case["scaling"] == "linear":
        f = f / s
    if case["scaling"] == "ramp":
        turns = _ORIGINAL_LENGTH * f / (2 * math.pi)
        keep = ((turns - _LOW) / (_HIGH - _LOW)).clamp(0, 1)
        f = f * (keep + (1 - keep) / s)
        magnitude = 1 + 0.1 * math.log(s)
    return f.to(_DEV), magnitude


def _plan(case, axes):
    return _package().RotaryPlan(case["turned"], axes=axes, interleaved=case["interleaved"],
                                 scaling=case["scaling"], factor=case["factor"], original_length=_ORIGINAL_LENGTH,
                                 low=_LOW, high=_HIGH)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _randn(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def randn(*shape):
        return torch.randn(shape, generator=g, device=_DEV, dtype=torch.float32).to(dtype)

    return randn, g


def _rotary_inputs(case, seed):
    randn, _ = _randn(case, seed)
    size, B, H, Hkv, D = _ints(case["size"]), case["batch"], case["heads"], case["kv_heads"], case["dim"]
    s = {}
    if case["packed"]:
        qkv = randn(B, *size, 3, H, D)
        s["q"], s["k"], _ = qkv.unbind(len(size) + 1)
    else:
        s["q"], s["k"] = randn(B, *size, H, D), randn(B, *size, Hkv, D)
    if case["grad"]:
        s["dq"], s["dk"] = randn(B, *size, H, D), randn(B, *size, Hkv, D)
    s["positions"] = None
    if len(size) == 1:
        # requests packed side by side continue at positions of their own
        at = case["start"] + torch.arange(B, device=_DEV)[:, None] * 1013
        s["positions"] = at + torch.arange(size[0], device=_DEV)
    return s


def _cache_inputs(case, seed):
    randn, g = _randn(case, seed)
    B, Hkv, D, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    rows = _lengths(case)
    # the same lengths in another order for another seed
    turn = seed % B
    rows = rows[turn:] + rows[:turn]
    s = {"new": [n for n, _ in rows], "lens": [n + c for n, c in rows]}
    per = [-(-n // page) for n in s["lens"]]
    pages = max(sum(per) + 3, 4)
    order = torch.randperm(pages, generator=g, device=_DEV, dtype=torch.int32)
    wide = max(max(per), 1)
    # pages lie anywhere in the pool; entries past a sequence's end name none
    used = torch.arange(wide, device=_DEV)[None] < torch.tensor(per, device=_DEV)[:, None]
    index = torch.tensor([sum(per[:b]) for b in range(B)], device=_DEV)[:, None] + torch.arange(wide, device=_DEV)
    s["table"] = torch.where(used, order[index.clamp(max=pages - 1)], -1).to(torch.int32)
    s["k_pages"], s["v_pages"] = randn(pages, page, Hkv, D), randn(pages, page, Hkv, D)
    s["seq_lens"] = torch.tensor(s["lens"], dtype=torch.int32, device=_DEV)
    s["new_lens"] = torch.tensor(s["new"], dtype=torch.int32, device=_DEV)
    s["q"] = randn(B, case["new"], case["heads"], D)
    if case["op"] == "append":
        s["k"], s["v"] = randn(B, case["new"], Hkv, D), randn(B, case["new"], Hkv, D)
    return s


def _inputs(case, seed):
    return _rotary_inputs(case, seed) if case["op"] == "rotary" else _cache_inputs(case, seed)


def prepare(case, seed):
    st = dict(_inputs(case, seed), op=case["op"], case=case)
    if case["op"] != "paged":
        axes = len(_ints(case["size"])) if case["op"] == "rotary" else 1
        if own:
            st["plan"] = _plan(case, axes)
        else:
            st["axes"] = axes
            st["freq"], st["magnitude"] = _frequencies(case, axes)
    if case["op"] == "rotary" and case["grad"]:
        st["leaves"] = [st["q"].detach().requires_grad_(True), st["k"].detach().requires_grad_(True)]
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _own_rotary(s):
    na = _package()
    if "leaves" not in s:
        return na.rotary_qk(s["q"], s["k"], s["plan"], s["positions"])
    q, k = na.rotary_qk(*s["leaves"], s["plan"], s["positions"])
    return (q, k, *torch.autograd.grad((q, k), s["leaves"], (s["dq"], s["dk"])))


def _own_append(s):
    q = _package().na1d_paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["seq_lens"],
                                     s["new_lens"], query=s["q"], plan=s["plan"])
    return q, s["k_pages"], s["v_pages"]


def _own_paged(s):
    c = s["case"]
    return _package().na1d_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["seq_lens"],
                                 c["kernel"] or None, c["dilation"], new_lens=s["new_lens"], return_lse=True)


def _grid(size):
    """Coordinates [*size, axes] of every position."""
    return torch.stack(torch.meshgrid(*(torch.arange(n, device=_DEV) for n in size), indexing="ij"), dim=-1)


def _turn(x, cos, sin, interleaved):
    """x [..., heads, dim] with each axis's share of its first dims turned;
    cos and sin [..., 1, axes, pairs]."""
    axes, pairs = cos.shape[-2:]
    turned = 2 * axes * pairs
    y = x.float()
    a = y[..., :turned].unflatten(-1, (axes, pairs, 2) if interleaved else (axes, 2, pairs))
    u, v = a.unbind(-1) if interleaved else a.unbind(-2)
    a = torch.stack((u * cos - v * sin, u * sin + v * cos), dim=-1 if interleaved else -2)
    return torch.cat((a.flatten(-3), y[..., turned:]), dim=-1).to(x.dtype)


def _cos_sin(s, coords):
    """cos and sin [..., 1, axes, pairs] of coordinates [..., axes]."""
    angle = coords[..., None].double() * s["freq"]
    m = s["magnitude"]
    return (angle.cos() * m).float().unsqueeze(-3), (angle.sin() * m).float().unsqueeze(-3)


def _plain_rotary(s):
    size = _ints(s["case"]["size"])
    coords = _grid(size) if s["positions"] is None else s["positions"][..., None]
    cos, sin = _cos_sin(s, coords)
    inter = s["case"]["interleaved"]
    out = (_turn(s["q"], cos, sin, inter), _turn(s["k"], cos, sin, inter))
    if "leaves" in s:
        # the gradient turns back by the same angles
        out += (_turn(s["dq"], cos, -sin, inter), _turn(s["dk"], cos, -sin, inter))
    return out


def _new_rows(s):
    """Sequence, token and position of every new token of the batch."""
    seq = torch.cat([torch.full((n,), b, device=_DEV) for b, n in enumerate(s["new"])])
    tok = torch.cat([torch.arange(n, device=_DEV) for n in s["new"]])
    pos = torch.cat([torch.arange(t - n, t, device=_DEV) for n, t in zip(s["new"], s["lens"])])
    return seq, tok, pos


def _plain_append(s):
    page = s["case"]["page"]
    seq, tok, pos = _new_rows(s)
    cos, sin = _cos_sin(s, pos[:, None])
    inter = s["case"]["interleaved"]
    at, slot = s["table"][seq, pos // page].long(), pos % page
    s["k_pages"][at, slot] = _turn(s["k"][seq, tok], cos, sin, inter)
    s["v_pages"][at, slot] = s["v"][seq, tok]
    q = torch.zeros_like(s["q"])
    q[seq, tok] = _turn(s["q"][seq, tok], cos, sin, inter)
    return q, s["k_pages"], s["v_pages"]


def _span(case, new, length):
    """First key that any of the new tokens attends to."""
    return max(0, length - new - (case["kernel"] - 1) * case["dilation"]) if case["kernel"] else 0


def _visible(case, queries, keys):
    """Which of the key positions each query position attends to."""
    back = queries[:, None] - keys[None]
    ok = back >= 0
    if case["kernel"]:
        ok &= (back < case["kernel"] * case["dilation"]) & (back % case["dilation"] == 0)
    return ok


def _plain_paged(s):
    c = s["case"]
    q, page, Hkv, D = s["q"], c["page"], c["kv_heads"], c["dim"]
    B, L, H, _ = q.shape
    out = torch.zeros_like(q)
    lse = torch.full((B, L, H), -math.inf, device=_DEV)
    for b, (n, length) in enumerate(zip(s["new"], s["lens"])):
        if n == 0:
            continue
        first = _span(c, n, length)
        keys = torch.arange(first, length, device=_DEV)
        at, slot = s["table"][b, keys // page].long(), keys % page
        hidden = ~_visible(c, torch.arange(length - n, length, device=_DEV), keys)
        for h in range(Hkv):
            heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
            k, v = s["k_pages"][at, slot, h].float(), s["v_pages"][at, slot, h].float()
            logits = (q[b, :n, heads].float() * D ** -0.5) @ k.t()          # [n, heads, keys]
            logits = logits.masked_fill(hidden[:, None], -math.inf)
            top = logits.amax(-1, keepdim=True)
            p = (logits - top).exp()
            total = p.sum(-1, keepdim=True)
            out[b, :n, heads] = ((p @ v) / total).to(q.dtype)
            lse[b, :n, heads] = (top + total.log())[..., 0]
    return out, lse


_own = {"rotary": _own_rotary, "append": _own_append, "paged": _own_paged}
_plain = {"rotary": _plain_rotary, "append": _plain_append, "paged": _plain_paged}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def _attended(case):
    """(query-key pairs, keys that some query attends to) over the batch, per
    kv head's group."""
    pairs = keys = 0
    K, d = case["kernel"], case["dilation"]
    for n, c in _lengths(case):
        if not K:
            pairs += n * c + n * (n + 1) // 2
            keys += c + n if n else 0
            continue
        for r in range(min(n, d)):
            # tokens r, r + d, ... share a residue class; member m of the
            # class is the query of member m's window
            members = (n - r + d - 1) // d
            first = (c + r) // d
            short = max(0, min(members, K - 1 - first))  # windows cut at the start
            pairs += members * K - sum(K - 1 - first - m for m in range(short))
            keys += min(first + members, members + K - 1)
    return pairs, keys


def work(case):
    esz = 4 if case["dtype"] == "float32" else 2
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        n = case["batch"] * math.prod(_ints(case["size"]))
        passes = 2 if case["grad"] else 1
        positions = 8 * n if len(_ints(case["size"])) == 1 else 0
        return {"bytes": float(passes * (2 * esz * n * (H + Hkv) * D + positions)),
                "flops": 3.0 * passes * n * (H + Hkv) * case["turned"]}
    new = sum(n for n, _ in _lengths(case))
    if case["op"] == "append":
        return {"bytes": float(2 * esz * new * (H + 2 * Hkv) * D), "flops": 3.0 * new * (H + Hkv) * case["turned"]}
    pairs, keys = _attended(case)
    return {"bytes": float(esz * D * (2 * new * H + 2 * keys * Hkv) + 4 * new * H), "flops": 4.0 * pairs * H * D}


# ---------------------------------------------------------------------------
# float64
# ---------------------------------------------------------------------------


def _exact_turn(x, coords, case, axes, back=False):
    """Each pair of a head as a complex number, times m * e^(i angle)."""
    f, m = _frequencies(case, axes)
    angle = coords.double()[..., None] * f                                  # [..., axes, pairs]
    factor = torch.polar(torch.full_like(angle, m), -angle if back else angle)[..., None, :, :]
    y, pairs = x.double().clone(), f.numel()
    for a in range(axes):
        lo = 2 * a * pairs
        if case["interleaved"]:
            one, two = slice(lo, lo + 2 * pairs, 2), slice(lo + 1, lo + 2 * pairs, 2)
        else:
            one, two = slice(lo, lo + pairs), slice(lo + pairs, lo + 2 * pairs)
        z = torch.complex(y[..., one], y[..., two]) * factor[..., a, :]
        y[..., one], y[..., two] = z.real, z.imag
    return y


def _exact_rotary(case, s):
    size = _ints(case["size"])
    coords = _grid(size) if s["positions"] is None else s["positions"][..., None]
    out = [_exact_turn(s[n], coords, case, len(size)) for n in ("q", "k")]
    if case["grad"]:
        out += [_exact_turn(s[n], coords, case, len(size), back=True) for n in ("dq", "dk")]
    return tuple(out)


def _exact_append(case, s):
    q, kp, vp = torch.zeros_like(s["q"], dtype=torch.float64), s["k_pages"].double(), s["v_pages"].double()
    P, page, Hkv, D = kp.shape
    for b, (n, length) in enumerate(zip(s["new"], s["lens"])):
        pos = torch.arange(length - n, length, device=_DEV)
        flat = s["table"][b].long().index_select(0, pos // page) * page + pos % page
        q[b, :n] = _exact_turn(s["q"][b, :n], pos[:, None], case, 1)
        kp.view(P * page, Hkv, D).index_copy_(0, flat, _exact_turn(s["k"][b, :n], pos[:, None], case, 1))
        vp.view(P * page, Hkv, D).index_copy_(0, flat, s["v"][b, :n].double())
    return q, kp, vp


def _exact_paged(case, s):
    B, L, H, D = s["q"].shape
    P, page, Hkv, _ = s["k_pages"].shape
    out = torch.zeros(B, L, H, D, dtype=torch.float64, device=_DEV)
    lse = torch.full((B, L, H), -math.inf, dtype=torch.float64, device=_DEV)
    for b, (n, length) in enumerate(zip(s["new"], s["lens"])):
        # blocks of queries, each over the keys from its first window on
        for i in range(0, n, 512):
            m = min(512, n - i)
            end = length - n + i + m
            keys = torch.arange(_span(case, m, end), end, device=_DEV)
            flat = s["table"][b].long().index_select(0, keys // page) * page + keys % page
            ok = _visible(case, torch.arange(end - m, end, device=_DEV), keys)
            bias = torch.zeros(ok.shape, dtype=torch.float64, device=_DEV).masked_fill_(~ok, -math.inf)
            for h in range(H):
                kv = h // (H // Hkv)
                k = s["k_pages"].view(P * page, Hkv, D)[flat, kv].double()
                v = s["v_pages"].view(P * page, Hkv, D)[flat, kv].double()
                logits = torch.addmm(bias, s["q"][b, i:i + m, h].double(), k.t(), alpha=D ** -0.5)
                lse[b, i:i + m, h] = logits.logsumexp(-1)
                out[b, i:i + m, h] = logits.softmax(-1) @ v
    return out, lse


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "paged": _exact_paged}[case["op"]](case, s)
