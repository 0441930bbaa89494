"""Beams whose logits have several of +infinity: their continuations share the row's weight and are compared in 64 bits as all others are."""
import math

import numpy as np
import pytest
import torch

from cachegen_b200 import paged
from pages_ref import best
from test_gpu_beams import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("turned", [False, True])
def test_counts_against_a_score_next_to_their_logarithm(dtype, turned):
    """Of a request's two beams one has n infinite logits, each of a share 1 / n, and the other a single one and a score that is -log n rounded to 32 bits."""
    vocab, counts = 1000, range(1, 1001)
    logits = torch.zeros((len(counts), 2, vocab), dtype=dtype, device="cuda")
    scores = torch.zeros((len(counts), 2), device="cuda")
    for i, n in enumerate(counts):
        logits[i, 0, (torch.arange(n, device="cuda") * 79 + i) % vocab] = math.inf  # (79 and the vocabulary have no factor in common)
        logits[i, 1, 11] = math.inf
        scores[i, 1] = -math.log(n)
    if turned:
        logits, scores = logits.flip(1), scores.flip(1)
    check(logits.reshape(-1, vocab), scores.contiguous(), 2)
    check(logits.reshape(-1, vocab), scores.contiguous(), 40)


def test_many_beams_of_the_same_infinite_logits():
    """More continuations alike than are sorted at once: the rows' heads are taken one by one."""
    logits = torch.full((64, 900), -math.inf, dtype=torch.float32, device="cuda")
    for i in range(64):
        logits[i, :300 + i] = math.inf
    scores = -torch.tensor([math.log(300.0) - math.log(300.0 + i) for i in range(64)], dtype=torch.float64).float().view(1, 64).cuda()
    got = paged.beam_select(logits, scores, 100)
    want = best(logits.cpu().numpy(), scores.cpu().numpy(), 100)
    assert np.array_equal(got[1].cpu().numpy(), want[1]) and np.array_equal(got[2].cpu().numpy(), want[2])
    assert (np.abs(got[0].cpu().numpy() - want[0]) <= 5e-6 + 2.0 ** -24 * np.abs(want[0])).all()
