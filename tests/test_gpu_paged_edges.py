"""Calls on a paged cache at the edges of what they allow: the widest windows, the most uneven weights, values that are not finite."""
import math

import pytest
import torch

from paged_ref import attention
from test_gpu_paged_attention import Batch, ids

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31, 2 ** 40])
@pytest.mark.parametrize("lens,heads", [([(16, 10)], 4), ([(5, 0), (3, 1), (4, 2)], 2), ([(20, 10), (40, 40)], 1), ([(300, 77), (150, 1)], 4)], ids=ids)
def test_windows_wider_than_any_context(lens, heads, window, causal):
    """More rows than keys, so that places are negative: such a window hides nothing."""
    b = Batch(lens, 4, heads, 64, 16, torch.float16)
    b.check(*b.call(window=window, causal=causal, max_q=max(n for n, _ in lens)), causal=causal)
