"""Causal 1-D neighbourhood attention over a paged cache of keys and values:
the serving form of ``na1d(..., is_causal=True)`` (no counterpart in the
reference).

Token ``j`` of sequence ``b`` lies at slot ``j % page_size`` of page
``block_table[b, j // page_size]``; pages are ``[pages, page_size, heads_kv,
dim]``.  ``seq_lens[b]`` counts the tokens of the sequence with the new ones
of this call, ``new_lens[b]`` (clamped to ``[0, L]``) the new ones: token ``i``
of the call's padded ``[B, L, heads, dim]`` tensors is at position
``seq_lens[b] - new_lens[b] + i``, so a call of fewer tokens than that holds
the last ones of the sequence.  Lengths and tables are device tensors and are never read back, so the
calls can be captured into a graph and replayed as the cache grows.

A table entry outside ``[0, pages)`` (like -1) names no page, nor does a
position past the table's width: tokens there are not written, and no query
attends to them.  A page that takes new tokens must belong to one sequence;
pages that are only read may be shared.

These calls have no gradients: they refuse tensors that need them, or carry
forward-mode tangents.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch

from natten_mps_amd._core import ops
from natten_mps_amd.positions import RotaryPlan, check_plan, has_tangent
from natten_mps_amd.utils.params import normalize_kernel_size, normalize_tuple_param

_INTS = (torch.int32, torch.int64)


def _hook(name: str):
    fn = getattr(ops.active_module(), name, None)
    if fn is None:
        raise NotImplementedError(f"backend '{ops.get_backend()}' has no paged cache.")
    return fn


def _call(name: str, x):
    """The backend's check and run of an ordinary call, where it has one."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        return None
    return getattr(ops.active_module(), name, None)


def _no_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradients: call it under torch.no_grad() or detach its tensors.")
    if has_tangent(*tensors):
        raise RuntimeError(f"{what} has no gradients: it takes no dual tensors (forward-mode differentiation).")


def _check_cache(what, batch, tokens, key_pages, value_pages, block_table, seq_lens, new_lens) -> None:
    if key_pages.ndim != 4 or value_pages.ndim != 4:
        raise ValueError(f"{what} expects pages with shape [pages, page_size, heads_kv, dim].")
    if key_pages.shape[:3] != value_pages.shape[:3]:
        raise ValueError(f"key and value pages must match but for their head dims: {tuple(key_pages.shape)}, "
                         f"{tuple(value_pages.shape)}.")
    if key_pages.numel() == 0 or value_pages.numel() == 0:
        raise ValueError("the cache must have at least one page of one token.")
    if key_pages.stride(-1) != 1 or value_pages.stride(-1) != 1:
        raise ValueError("pages must be contiguous in their head dim.")
    if block_table.ndim != 2 or block_table.shape[0] != batch or block_table.shape[1] < 1:
        raise ValueError(f"block_table must be [B={batch}, pages of a sequence], got {tuple(block_table.shape)}.")
    for name, t in (("seq_lens", seq_lens), ("new_lens", new_lens)):
        if t is not None and tuple(t.shape) != (batch,):
            raise ValueError(f"{name} must be a 1-D tensor of length B={batch}, got shape {tuple(t.shape)}.")
    for name, t in (("block_table", block_table), ("seq_lens", seq_lens), ("new_lens", new_lens)):
        if t is not None and t.dtype not in _INTS:
            raise ValueError(f"{name} must be int32 or int64, got {t.dtype}.")


def na1d_paged_append(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                      block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: Optional[torch.Tensor] = None,
                      *, query: Optional[torch.Tensor] = None,
                      plan: Optional[RotaryPlan] = None) -> Optional[torch.Tensor]:
    """Write the new tokens' ``key [B, L, heads_kv, dim]`` and ``value`` to
    their pages, in place.

    With a ``plan`` (of one axis) the keys are turned by their positions on
    the way, and so is ``query [B, L, heads, dim]`` when given: the result,
    a new tensor with zeros at padding tokens (without a plan, the query's
    values).  Returns None without a query.  Other slots of the pages, and
    those of padding tokens, stay as they are; ``key`` and ``value`` must not
    overlap the pages."""
    fn = _call("paged_append_call", key)
    if fn is not None and (plan is None or type(plan) is RotaryPlan):
        done = fn(key, value, key_pages, value_pages, block_table, seq_lens, new_lens, query, plan)
        if done is not None:
            return done[0] if done else None
    what = "na1d_paged_append"
    if key.ndim != 4 or value.ndim != 4 or key.shape[:3] != value.shape[:3]:
        raise ValueError(f"{what} expects key and value with shape [B, L, heads_kv, dim], matching but for their "
                         f"head dims: {tuple(key.shape)}, {tuple(value.shape)}.")
    batch, tokens = key.shape[:2]
    _check_cache(what, batch, tokens, key_pages, value_pages, block_table, seq_lens, new_lens)
    if key.shape[2:] != key_pages.shape[2:] or value.shape[2:] != value_pages.shape[2:]:
        raise ValueError(f"key and value heads and dims must be those of the pages: {tuple(key.shape[2:])}, "
                         f"{tuple(value.shape[2:])}; {tuple(key_pages.shape[2:])}, {tuple(value_pages.shape[2:])}.")
    for name, t in (("key_pages", key_pages), ("value_pages", value_pages)):
        if any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape)):
            raise ValueError(f"{name} is written and cannot be an expanded tensor.")
    if query is not None and (query.ndim != 4 or query.shape[:2] != key.shape[:2] or query.shape[-1] != key.shape[-1]):
        raise ValueError(f"query must be [B, L, heads, dim] like key but for its heads: {tuple(query.shape)}, "
                         f"{tuple(key.shape)}.")
    if plan is not None:
        check_plan(plan, key.shape[-1])
        if plan.axes != 1:
            raise ValueError(f"a cache has one axis of positions; the plan has {plan.axes}.")
    _no_grad(what, key, value, query, key_pages, value_pages)
    return _hook("paged_append")(key, value, key_pages, value_pages, block_table, seq_lens, new_lens, query, plan)


def na1d_paged(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor, block_table: torch.Tensor,
               seq_lens: torch.Tensor, kernel_size: Union[int, Tuple[int], None] = None,
               dilation: Union[int, Tuple[int]] = 1, *, new_lens: Optional[torch.Tensor] = None,
               scale: Optional[float] = None, return_lse: bool = False):
    """Attention of the new tokens' ``query [B, L, heads, dim]`` over the
    paged cache (which holds their own keys already).

    The query at position ``p`` attends to the keys ``p - t * dilation >= 0``,
    ``t < kernel_size``: what ``na1d(..., is_causal=True)`` over the whole
    sequence gives for its last tokens.  ``kernel_size`` None: all keys
    ``0..p``.  Query head ``h`` reads kv head ``h // (heads / heads_kv)``.
    Returns ``[B, L, heads, dim_v]``, or ``(out, lse)`` with ``lse [B, L,
    heads]`` in float32 when ``return_lse`` (with which
    :func:`~natten_mps_amd.merge_attentions` adds other keys).  Padding
    tokens, and queries without a key, have zeros and an lse of -inf."""
    fn = _call("paged_forward_call", query)
    if fn is not None:
        done = fn(query, key_pages, value_pages, block_table, seq_lens, new_lens, kernel_size, dilation, scale)
        if done is not None:
            return done if return_lse else done[0]
    what = "na1d_paged"
    if query.ndim != 4:
        raise ValueError(f"{what} expects query with shape [B, L, heads, dim], got {tuple(query.shape)}.")
    batch, tokens, heads, dim = query.shape
    _check_cache(what, batch, tokens, key_pages, value_pages, block_table, seq_lens, new_lens)
    if dim != key_pages.shape[-1]:
        raise ValueError(f"Head dim must match between query and key pages: {dim}, {key_pages.shape[-1]}.")
    if heads < 1 or heads % key_pages.shape[2] != 0:
        raise ValueError(f"heads_q ({heads}) must be divisible by heads_kv ({key_pages.shape[2]}) for GQA.")
    ks = None if kernel_size is None else normalize_kernel_size(kernel_size, 1)[0]
    dil = normalize_tuple_param(dilation, 1, "dilation")[0]
    if isinstance(dil, bool):
        raise ValueError("dilation must contain integers, not bools.")
    if ks is None and dil != 1:
        raise ValueError("a dilation needs a kernel_size.")
    _no_grad(what, query, key_pages, value_pages)
    out, lse = _hook("paged_forward")(query, key_pages, value_pages, block_table, seq_lens, new_lens, ks, dil,
                                      dim ** -0.5 if scale is None else float(scale))
    return (out, lse) if return_lse else out


class PagedKVCache:
    """Pages of keys and values for a batch of sequences, and which sequence
    holds which page.

    ``layers`` attention layers share the lengths and the table; layer ``i``
    (:meth:`layer`) has pages of its own.  A step of a program::

        cache.reserve(new_tokens)              # pages for the next tokens
        for i, attn in enumerate(layers):      # NeighborhoodAttention1D
            x = x + attn(x, cache=cache.layer(i))

    :meth:`reserve` does its bookkeeping on the host and sends the changed
    lengths and tables to the device on the current stream without waiting;
    the device tensors (``block_table``, ``seq_lens``, ``new_lens``) keep
    their addresses, so a captured step can be replayed after it.  It belongs
    between the replays: neither it nor :meth:`release` and :meth:`trim` can
    be captured.
    """

    def __init__(self, num_pages: int, page_size: int, batch: int, num_kv_heads: int, head_dim: int, *,
                 value_dim: Optional[int] = None, max_pages: Optional[int] = None, layers: int = 1,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        value_dim = head_dim if value_dim is None else value_dim
        max_pages = num_pages if max_pages is None else max_pages
        for name, n in (("num_pages", num_pages), ("page_size", page_size), ("batch", batch),
                        ("num_kv_heads", num_kv_heads), ("head_dim", head_dim), ("value_dim", value_dim),
                        ("max_pages", max_pages), ("layers", layers)):
            if isinstance(n, bool) or not isinstance(n, int) or n < 1:
                raise ValueError(f"{name} must be an integer >= 1, got {n!r}.")
        self.num_pages, self.page_size, self.batch, self.max_pages = num_pages, page_size, batch, max_pages
        self.layers = layers
        self.device = torch.device(device)
        shape = (layers, num_pages, page_size, num_kv_heads)
        self.key_pages = torch.zeros(*shape, head_dim, dtype=dtype, device=self.device)
        self.value_pages = torch.zeros(*shape, value_dim, dtype=dtype, device=self.device)
        # one device buffer: lengths, new lengths, table
        self._rows = 2 * batch
        self._meta = torch.zeros(self._rows + batch * max_pages, dtype=torch.int32, device=self.device)
        self._meta[self._rows:] = -1
        self.seq_lens, self.new_lens = self._meta[:batch], self._meta[batch:self._rows]
        self.block_table = self._meta[self._rows:].view(batch, max_pages)
        self._free = list(range(num_pages - 1, -1, -1))
        self._tables: List[List[int]] = [[] for _ in range(batch)]
        self._lens = [0] * batch
        self._new = [0] * batch

    @property
    def lengths(self) -> List[int]:
        """Tokens of each sequence, as the host counts them."""
        return list(self._lens)

    @property
    def new_tokens(self) -> int:
        """New tokens of a sequence, at most, that the last :meth:`reserve`
        made room for."""
        return max(self._new)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def layer(self, index: int) -> "PagedLayer":
        if not 0 <= index < self.layers:
            raise IndexError(f"layer {index} of {self.layers}.")
        return PagedLayer(self, index)

    def _index(self, sequence: int) -> int:
        if not 0 <= sequence < self.batch:
            raise IndexError(f"sequence {sequence} of {self.batch}.")
        return sequence

    def _host_step(self, what: str) -> None:
        # a replay would send what the host's memory holds by then
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"PagedKVCache.{what} cannot be captured into a graph: call it between replays.")

    def reserve(self, new_tokens: Union[int, Sequence[int]]) -> None:
        """Make room for the next ``new_tokens`` of each sequence (one number
        for all, or one each, 0 for a sequence that waits) and count them as
        the new tokens of the calls that follow.  Raises RuntimeError, and
        changes nothing, where pages run out."""
        self._host_step("reserve")
        counts = [new_tokens] * self.batch if isinstance(new_tokens, int) else list(new_tokens)
        if len(counts) != self.batch or any(isinstance(n, bool) or not isinstance(n, int) or n < 0 for n in counts):
            raise ValueError(f"new_tokens must be a count >= 0 for each of the {self.batch} sequences.")
        need = [max(-(-(len_ + n) // self.page_size) - len(t), 0)
                for len_, n, t in zip(self._lens, counts, self._tables)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {sum(need)} pages needed, {len(self._free)} free.")
        for b, (t, n) in enumerate(zip(self._tables, need)):
            if len(t) + n > self.max_pages:
                raise RuntimeError(f"PagedKVCache: sequence {b} needs {len(t) + n} pages, at most {self.max_pages}.")
        changed = []
        for b, (t, n) in enumerate(zip(self._tables, need)):
            for _ in range(n):
                changed.append((self._entry(b, len(t)), self._free[-1]))
                t.append(self._free.pop())
        self._lens = [a + n for a, n in zip(self._lens, counts)]
        self._new = counts
        self._send(changed)

    def release(self, sequence: int) -> None:
        """Give a sequence's pages back; it starts again at length 0."""
        self._host_step("release")
        b = self._index(sequence)
        changed = [(self._entry(b, i), -1) for i, p in enumerate(self._tables[b]) if p >= 0]
        self._free.extend(p for p in reversed(self._tables[b]) if p >= 0)
        self._tables[b] = []
        self._lens[b] = self._new[b] = 0
        self._send(changed)

    def trim(self, kernel_size: int, dilation: int = 1) -> None:
        """Give back the pages that lie wholly behind the windows of every
        token to come (attention with this or a smaller ``kernel_size`` and
        ``dilation``); their table entries become -1.  Call it after the
        step's attention: the new tokens' own windows may reach further back."""
        self._host_step("trim")
        ks = normalize_kernel_size(kernel_size, 1)[0]
        reach = (ks - 1) * normalize_tuple_param(dilation, 1, "dilation")[0]
        changed = []
        for b, (t, n) in enumerate(zip(self._tables, self._lens)):
            for i in range(min(max(n - reach, 0) // self.page_size, len(t))):
                if t[i] >= 0:
                    self._free.append(t[i])
                    t[i] = -1
                    changed.append((self._entry(b, i), -1))
        if changed:
            self._send(changed)

    def _entry(self, sequence: int, index: int) -> int:
        """Where in the device buffer an entry of a sequence's table lies."""
        return self._rows + sequence * self.max_pages + index

    def _send(self, changed: List[Tuple[int, int]]) -> None:
        """Lengths, and the table's entries that changed, to the device."""
        pin = self.device.type == "cuda"
        host = torch.tensor(self._lens + self._new, dtype=torch.int32, pin_memory=pin)
        self._meta[:self._rows].copy_(host, non_blocking=pin)
        if changed:
            pairs = torch.tensor(changed, dtype=torch.int64, pin_memory=pin).to(self.device, non_blocking=pin)
            self._meta.index_copy_(0, pairs[:, 0], pairs[:, 1].to(torch.int32))


class PagedLayer:
    """One layer's pages of a :class:`PagedKVCache`."""

    def __init__(self, cache: PagedKVCache, index: int):
        self.cache = cache
        self.key_pages, self.value_pages = cache.key_pages[index], cache.value_pages[index]

    def append(self, key, value, *, query=None, plan=None):
        """:func:`na1d_paged_append` of the reserved tokens."""
        c = self.cache
        return na1d_paged_append(key, value, self.key_pages, self.value_pages, c.block_table, c.seq_lens, c.new_lens,
                                 query=query, plan=plan)

    def attend(self, query, kernel_size=None, dilation=1, *, scale=None, return_lse=False):
        """:func:`na1d_paged` of the reserved tokens."""
        c = self.cache
        return na1d_paged(query, self.key_pages, self.value_pages, c.block_table, c.seq_lens, kernel_size, dilation,
                          new_lens=c.new_lens, scale=scale, return_lse=return_lse)


__all__ = ["PagedKVCache", "PagedLayer", "na1d_paged", "na1d_paged_append"]
