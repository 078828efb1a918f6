"""Rotary positions for queries and keys (no counterpart in the reference).

A pair ``(u, v)`` of a head at coordinate ``x`` turns by the angle
``t = x * f`` of its frequency: ``(u', v') = m (u cos t - v sin t,
u sin t + v cos t)``.  :class:`RotaryPlan` holds the frequencies, which dims
turn and how they pair; :func:`rotary` and :func:`rotary_qk` turn tensors in
the package's layout ``[B, *spatial, heads, dim]``, with gradients (the map's
transpose, the same turn backwards) and forward-mode tangents.

On a grid each axis owns an equal share of the turned dims, and a token's
coordinates are its indices::

    plan = RotaryPlan(48, axes=3)             # 16 dims per axis, dims 48.. stay
    q, k = rotary_qk(q, k, plan)              # [B, D, H, W, heads, 64]
    out = na3d(q, k, v, kernel_size=(3, 7, 7))

Angles hold at any position: a frequency is kept as the nearest 64-bit
fraction of a turn, and its product with an integer position ``p`` drops whole
turns without rounding, so the angle is off by ``2^-65 |p|`` turns at most.
"""
from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from natten_mps_amd._core import ops

_SCALINGS = ("none", "linear", "base", "ramp")


def _number(value, name: str) -> float:
    if isinstance(value, bool) or not isinstance(value, (int, float)) or not math.isfinite(value):
        raise ValueError(f"{name} must be a finite number, got {value!r}.")
    return float(value)


@lru_cache(maxsize=None)
def _pi(bits: int) -> int:
    """pi 2^bits, to a unit or two: Machin's 16 atan(1/5) - 4 atan(1/239)."""
    one = 1 << (bits + 16)

    def atan_inverse(x):
        total = term = one // x
        n, sign = 3, -1
        while term:
            term //= x * x
            total += sign * (term // n)
            n, sign = n + 2, -sign
        return total

    return (16 * atan_inverse(5) - 4 * atan_inverse(239)) >> 16


def _turn_fraction(f: float) -> int:
    """The float f, taken as it is, in turns times 2^64, to the nearest
    integer: f / (2 pi) in integers, with bits of pi for f's own size."""
    n, d = f.as_integer_ratio()
    bits = 80 + max(math.frexp(f)[1], 0)
    num, den = n << (64 + bits), 2 * d * _pi(bits)
    return (2 * num + den) // (2 * den)


class RotaryPlan:
    """Which dims of a head turn, how they pair, and by which frequencies.

    Args:
        dim: dims of the head that turn (its first ones), a multiple of
            ``2 * axes``; the rest passes through.
        axes: axes of positions (1..3); axis ``a`` owns the dims
            ``[a n, (a + 1) n)``, ``n = dim / axes``, and turns them as a
            plan of one axis would.
        interleaved: pairs are neighbours ``(2j, 2j + 1)``; otherwise
            ``(j, j + n / 2)``.
        base: frequencies ``base ** (-2 j / n)`` (angle per position of pair
            ``j``).
        scaling: for contexts ``factor`` times longer than trained on:

            * ``"none"``;
            * ``"linear"``: every frequency divided by ``factor``;
            * ``"base"``: the base multiplied by ``factor ** (n / (n - 2))``,
              so that the slowest frequency is divided by ``factor`` and the
              fastest one stays;
            * ``"ramp"``: a pair that makes ``r`` turns over
              ``original_length`` keeps its frequency where ``r >= high``,
              has it divided by ``factor`` where ``r <= low``, and a linear
              blend between.
        magnitude: factor on the turned dims; by default
            ``1 + 0.1 ln(factor)`` with ``"ramp"``, else 1.
        frequencies: explicit angles per position of the ``n / 2`` pairs of
            an axis, in place of ``base`` and ``scaling``.

    Plans are immutable and compare by value.
    """

    __slots__ = ("dim", "axes", "interleaved", "magnitude", "frequencies", "_turns", "_tables")

    def __init__(self, dim: int, *, axes: int = 1, interleaved: bool = False, base: float = 10000.0,
                 scaling: str = "none", factor: float = 1.0, original_length: Optional[int] = None,
                 low: float = 1.0, high: float = 32.0, magnitude: Optional[float] = None,
                 frequencies: Optional[Sequence[float]] = None):
        if isinstance(axes, bool) or not isinstance(axes, int) or not 1 <= axes <= 3:
            raise ValueError(f"axes must be 1, 2 or 3, got {axes!r}.")
        if isinstance(dim, bool) or not isinstance(dim, int) or dim <= 0 or dim % (2 * axes):
            raise ValueError(f"dim must be a positive multiple of 2 * axes ({2 * axes}), got {dim!r}.")
        if scaling not in _SCALINGS:
            raise ValueError(f"scaling must be one of {_SCALINGS}, got {scaling!r}.")
        n = dim // axes
        s = _number(factor, "factor")
        if s <= 0:
            raise ValueError(f"factor must be > 0, got {factor}.")
        if frequencies is not None:
            if scaling != "none":
                raise ValueError("frequencies cannot be combined with a scaling.")
            f = [_number(x, "frequencies") for x in frequencies]
            if len(f) != n // 2:
                raise ValueError(f"frequencies must hold one angle per pair of an axis ({n // 2}), got {len(f)}.")
        else:
            b = _number(base, "base")
            if b <= 0:
                raise ValueError(f"base must be > 0, got {base}.")
            if scaling == "base" and n > 2:
                b *= s ** (n / (n - 2))
            f = [b ** (-2 * j / n) for j in range(n // 2)]
            if scaling == "linear":
                f = [x / s for x in f]
            elif scaling == "ramp":
                if original_length is None or _number(original_length, "original_length") <= 0:
                    raise ValueError("scaling='ramp' needs the original_length (> 0).")
                lo, hi = _number(low, "low"), _number(high, "high")
                if not lo < hi:
                    raise ValueError(f"low ({low}) must be below high ({high}).")
                keep = [min(max((original_length * x / (2 * math.pi) - lo) / (hi - lo), 0.0), 1.0) for x in f]
                f = [x * (g + (1 - g) / s) for x, g in zip(f, keep)]
        if magnitude is None:
            magnitude = 1 + 0.1 * math.log(s) if scaling == "ramp" else 1.0
        # turns per position modulo 1, as 64-bit fractions (two's complement,
        # as torch's signed integers hold them)
        turns = [(_turn_fraction(x) + 2 ** 63) % 2 ** 64 - 2 ** 63 for x in f]
        for name, value in (("dim", dim), ("axes", axes), ("interleaved", bool(interleaved)),
                            ("magnitude", _number(magnitude, "magnitude")), ("frequencies", tuple(f)),
                            ("_turns", tuple(turns)), ("_tables", {})):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError("RotaryPlan is immutable.")

    def _key(self):
        return self.dim, self.axes, self.interleaved, self.magnitude, self.frequencies

    def __eq__(self, other):
        return isinstance(other, RotaryPlan) and self._key() == other._key()

    def __hash__(self):
        return hash(self._key())

    def __repr__(self):
        return (f"RotaryPlan({self.dim}, axes={self.axes}, interleaved={self.interleaved}, "
                f"magnitude={self.magnitude:g})")

    def __copy__(self):
        return self

    def __deepcopy__(self, memo):
        return self

    def __reduce__(self):
        return _restore, self._key()

    def table(self, device) -> torch.Tensor:
        """The frequencies on ``device``, one int64 per pair of an axis.  Made
        on the first call there (a copy that waits for the device, so not
        during graph capture) and kept until the process ends, but for those
        that a trace makes (fake tensors, or a compiled graph's own)."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        t = self._tables.get(device)
        if t is None:
            key = (device, self._turns)
            t = _TABLES.get(key)
            if t is None:
                if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("RotaryPlan: call plan.table(device) once before a graph is captured.")
                t = torch.tensor(self._turns, dtype=torch.int64).to(device)
                if type(t) is not torch.Tensor or torch.compiler.is_compiling():
                    return t
                _TABLES[key] = t
            self._tables[device] = t
        return t


# Tables by their values: a plan that goes while kernels of another stream
# still read its table must not give the memory back.
_TABLES: dict = {}


def _restore(dim, axes, interleaved, magnitude, frequencies):
    return RotaryPlan(dim, axes=axes, interleaved=interleaved, magnitude=magnitude, frequencies=frequencies)


def _check_tensor(x, name: str) -> None:
    if not isinstance(x, torch.Tensor) or x.ndim not in (4, 5, 6):
        raise ValueError(f"rotary expects {name} with shape [B, *spatial, heads, dim] (1 to 3 spatial axes).")


def check_plan(plan, dim: int) -> None:
    if not isinstance(plan, RotaryPlan):
        raise TypeError(f"plan must be a RotaryPlan, got {type(plan).__name__}.")
    if plan.dim > dim:
        raise ValueError(f"the plan turns {plan.dim} dims, the head has {dim}.")


def _check_positions(positions, plan, shape) -> None:
    sp = tuple(shape[1:-2])
    if positions is None:
        if plan.axes != len(sp):
            raise ValueError(f"a plan of {plan.axes} axes needs explicit positions on {len(sp)} spatial axes.")
        return
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}.")
    tail = () if plan.axes == 1 else (plan.axes,)
    got = tuple(positions.shape)
    if got not in (sp + tail, (1,) + sp + tail, (shape[0],) + sp + tail):
        raise ValueError(f"positions must have shape {sp + tail} or {(shape[0],) + sp + tail}, got {got}.")


class _RotaryFunction(torch.autograd.Function):
    """Turn by the positions' angles (backwards when ``inverse``); the
    gradient is the opposite turn, through this Function again, a tangent
    turns as the tensor does."""

    @staticmethod
    def forward(ctx, hook, plan, positions, inverse, *tensors):
        ctx.set_materialize_grads(False)
        ctx.hook, ctx.plan, ctx.inverse = hook, plan, inverse
        ctx.like = [(t.shape, t.dtype, t.device) for t in tensors]
        ctx.explicit = positions is not None
        if ctx.explicit:
            ctx.save_for_backward(positions)
            ctx.save_for_forward(positions)
        return tuple(hook(*tensors, *(None,) * (2 - len(tensors)), plan, positions, inverse)[:len(tensors)])

    @staticmethod
    def backward(ctx, *grads):
        positions = ctx.saved_tensors[0] if ctx.explicit else None
        given = [g for g in grads if g is not None]
        if given:
            given = list(_RotaryFunction.apply(ctx.hook, ctx.plan, positions, not ctx.inverse, *given))
        return (None, None, None, None, *(None if g is None else given.pop(0) for g in grads))

    @staticmethod
    def jvp(ctx, _hook, _plan, _positions, _inverse, *tangents):
        positions = ctx.saved_tensors[0] if ctx.explicit else None
        given = [t for t in tangents if t is not None]
        given = list(_turn(ctx.hook, ctx.plan, positions, ctx.inverse, *given))
        # autograd wants a tangent of each output
        return tuple(torch.zeros(shape, dtype=dtype, device=device) if t is None else given.pop(0)
                     for t, (shape, dtype, device) in zip(tangents, ctx.like))


def has_tangent(*tensors) -> bool:
    """Whether one of the tensors (None: absent) is a dual tensor of
    forward-mode differentiation."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _hook():
    mod = ops.active_module()
    fn = getattr(mod, "rotary", None)
    if fn is None:
        raise NotImplementedError(f"backend '{ops.get_backend()}' has no rotary positions.")
    return fn


def _call(x, key, plan, positions):
    """An ordinary call, checked and run by the backend; None otherwise."""
    if type(plan) is not RotaryPlan or not isinstance(x, torch.Tensor) or not x.is_cuda:
        return None
    fn = getattr(ops.active_module(), "rotary_call", None)
    return None if fn is None else fn(x, key, plan, positions)


def _turn(hook, plan, positions, inverse, *tensors):
    if (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)) or has_tangent(*tensors):
        return _RotaryFunction.apply(hook, plan, positions, inverse, *tensors)
    return hook(*tensors, *(None,) * (2 - len(tensors)), plan, positions, inverse)[:len(tensors)]


def rotary(x: torch.Tensor, plan: RotaryPlan, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` ``[B, *spatial, heads, dim]`` turned by the angles of its
    positions, a new tensor.

    ``positions``: None for the tokens' own indices (one plan axis per
    spatial axis), or int32 / int64 ``[*spatial]`` or ``[B, *spatial]``, with
    a trailing dim of coordinates when the plan has several axes."""
    done = _call(x, None, plan, positions)
    if done is not None:
        return done[0]
    _check_tensor(x, "a tensor")
    check_plan(plan, x.shape[-1])
    _check_positions(positions, plan, x.shape)
    return _turn(_hook(), plan, positions, False, x)[0]


def rotary_qk(query: torch.Tensor, key: torch.Tensor, plan: RotaryPlan,
              positions: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`rotary` of queries and keys in one launch; they may differ in
    their number of heads only."""
    done = _call(query, key, plan, positions)
    if done is not None:
        return done
    _check_tensor(query, "query")
    _check_tensor(key, "key")
    if query.shape[:-2] != key.shape[:-2] or query.shape[-1] != key.shape[-1]:
        raise ValueError(f"query and key must match but for their heads: {tuple(query.shape)}, {tuple(key.shape)}.")
    check_plan(plan, query.shape[-1])
    _check_positions(positions, plan, query.shape)
    return tuple(_turn(_hook(), plan, positions, False, query, key))


__all__ = ["RotaryPlan", "rotary", "rotary_qk"]
