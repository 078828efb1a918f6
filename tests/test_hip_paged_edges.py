"""Attention over a paged cache where its arithmetic has edges: windows of any
length beside tokens before the sequence.  Tolerances are those of
``test_hip_paged``."""
from __future__ import annotations

import pytest
import torch

from test_hip_paged import BF, DEV, F32, Problem, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hq, hkv, dim, dil", [(2, 2, 64, 1), (8, 2, 64, 1), (2, 2, 128, 2), (8, 2, 32, 2), (2, 1, 20, 1)])
@pytest.mark.parametrize("kernel", [2 ** 31 - 1, 2 ** 31 - 5])
def test_window_past_all_with_tokens_before_the_sequence(hq, hkv, dim, dil, kernel, dtype):
    """A window of any length over a sequence shorter than its new tokens:
    the tokens before position 0 are empty, the others see what there is."""
    p = Problem([(40, 40), (40, 40)], hq, hkv, dim, 16, dtype)
    p.lens = torch.tensor([30, 1], dtype=torch.int32, device=DEV)
    check(p.run(kernel, dil), p, kernel, dil)
