"""The paged cache around captured graphs."""
from __future__ import annotations

import pytest
import torch

import natten_mps_amd as na

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("call", [lambda c: c.reserve(1), lambda c: c.release(0), lambda c: c.trim(2)])
def test_bookkeeping_is_not_captured(call):
    """A captured copy would send, at each replay, whatever its host memory
    holds by then."""
    c = na.PagedKVCache(8, 4, 2, 1, 32, device=DEV)
    c.reserve([9, 3])
    state = (c.lengths, c.free_pages, c.block_table.clone(), c.seq_lens.clone())
    x = torch.zeros(4, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            x.add_(1)
            call(c)
    assert (c.lengths, c.free_pages) == state[:2]
    assert torch.equal(c.block_table, state[2]) and torch.equal(c.seq_lens, state[3])
    call(c)
