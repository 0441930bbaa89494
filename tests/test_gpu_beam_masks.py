"""The best continuations of beams whose logits are masked by a large finite number, as banned tokens are where -infinity is not wanted.

What is masked weighs exp(-2e4) of the rest at most, which is nothing: a score is off by what test_gpu_beams.py derives, the rounding to 32 bits and 5e-6."""
import numpy as np
import pytest
import torch

from cachegen_b200 import paged
from pages_ref import best
from test_gpu_beams import begun, check, rows

pytestmark = pytest.mark.gpu

MASKS = [(t, m) for t in (torch.float32, torch.bfloat16) for m in (-4e4, -1e6, -1e9, -2e9, -1e10, -1e12, -1e15, -1e20, -1e30, -1e32, -1e38, -2.3e38)] + [
    (torch.float16, m) for m in (-3e4, -4e4, -6e4)]


def masked(logits, mask, how, seed=0):
    """logits with `mask` in every second row, at the places that `how` names"""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, vocab = logits.shape
    token, per = torch.arange(vocab, device="cuda"), 16 // logits.element_size()
    if isinstance(how, float):
        where = torch.rand((n, vocab), generator=g, device="cuda") < how
    else:
        where = {"all but some": lambda: torch.ones((n, vocab), device="cuda").scatter_(1, torch.randint(0, vocab, (n, 50), generator=g, device="cuda"), 0.0) > 0,
                 "one thread": lambda: ((token // per % 256) == 77).expand(n, vocab), "one warp": lambda: ((token // per % 256) // 32 == 2).expand(n, vocab),
                 "behind the beginning": lambda: (token >= 1024 * per - 100).expand(n, vocab), "the beginning": lambda: (token < vocab - 60).expand(n, vocab),
                 "the middle": lambda: ((token > 40) & (token < vocab - 40)).expand(n, vocab)}[how]()
    out = logits.clone()
    out[::2] = torch.where(where[::2], torch.full_like(logits[::2], mask), logits[::2])
    return out


HOW = [0.5, 0.9, 0.99, "all but some", "one thread", "one warp", "behind the beginning", "the beginning", "the middle"]


@pytest.mark.parametrize("dtype,mask", MASKS)
def test_masked(dtype, mask):
    for vocab in (9000, 32000):
        logits = rows(4, vocab, dtype, vocab)
        for n, how in enumerate(HOW):
            x = masked(logits, mask, how, n)
            check(x, begun(1, 4, n), 16)  # several beams: a wrong sum changes which is chosen
            check(x, begun(4, 1, n), 64)  # more than are left of some rows


@pytest.mark.parametrize("dtype,mask", MASKS)
def test_the_mask_added(dtype, mask):
    """Logits plus the mask: banned ones are unlike, as far as the type can tell them apart, and still weigh nothing."""
    logits = rows(4, 20000, dtype, 3)
    check(torch.where(masked(logits, 1e9 if dtype != torch.float16 else 6e4, 0.97) == logits, logits, (logits.float() + mask).to(dtype)), begun(2, 2, 2), 20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_masks_and_rows_that_are_all_masked(dtype):
    for low, lower in ((-1e10, -1e20), (-2e9, -1e38), (-1e30, float("-inf")), (-1e15, torch.finfo(dtype).min)):
        x = masked(masked(rows(4, 15000, dtype, 5), low, 0.98), lower, 0.5, 1)
        x[2] = low
        x[2, 7000:] = lower
        x[3, :10000] = lower  # a part of a row without anything else
        check(x, begun(4, 1, 1), 9)
        check(x[[0, 1, 3]], begun(1, 3, 2), 9)


@pytest.mark.parametrize("dtype,requests,beams,vocab,k", [(torch.bfloat16, 64, 8, 128000, 16), (torch.float32, 16, 16, 65537, 32), (torch.float32, 40, 16, 66000, 16)])
@pytest.mark.parametrize("how", [0.9, "all but some", "behind the beginning"])
def test_a_batch(dtype, requests, beams, vocab, k, how):
    """Parts of many tiles, and those that lie across the ends of rows."""
    logits, scores = masked(rows(requests * beams, vocab, dtype, vocab), -1e10, how), begun(requests, beams, 7)
    got = [t.cpu().numpy() for t in paged.beam_select(logits, scores, k)]
    for b in (0, requests // 2, requests - 1):
        want = best(logits[b * beams:(b + 1) * beams].float().cpu().numpy(), scores[b:b + 1].cpu().numpy(), k)
        assert np.array_equal(got[1][b], want[1][0]) and np.array_equal(got[2][b], want[2][0] + b * beams)
        assert (np.abs(got[0][b] - want[0][0]) <= 5e-6 + 2.0 ** -24 * np.abs(want[0][0])).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_logits_on_both_sides_of_what_is_summed_the_quick_way(dtype):
    """Around -32,768, below which a thread's or a part's logits are summed otherwise, and 32,768."""
    for vocab in (9000, 70001):
        for spread in (2.0, 100.0):
            for middle in (-32768.0, 32768.0):
                x = (rows(4, vocab, torch.float32, vocab, spread=spread) + middle).to(dtype)
                check(x, begun(1, 4, 1), 8)
                check(masked(x, -6e4 if dtype == torch.float16 else -1e10, 0.98, 1), begun(2, 2, 1), 8)
                x[:, ::3] = -32768.0
                check(x, begun(4, 1, 1), 8)
