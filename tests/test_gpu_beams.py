"""The best continuations of beams against the same by its definition in 64 bits.

Tokens and parents are equal.  A score is off by the rounding to 32 bits, half a step or 2^-24 of itself, and by the error of a sum of exponentials in
32 bits, which enters as a logarithm: below 5e-6 whatever the logits (a term exp(-u) is off by 2^-24 (u + 6.3) + 1.4e-8 u and 2^-22, u weighted with the terms is
below 17 for 2^24 tokens, the 34 additions of a part's sum add 2^-24 each, and joining the parts 2^-21 and 2^-23)."""
import numpy as np
import pytest
import torch

from cachegen_b200 import paged
from pages_ref import best

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]
INF = float("inf")


def check(logits, scores, k):
    got = paged.beam_select(logits, scores, k)
    want = best(logits.float().cpu().numpy(), scores.cpu().numpy(), k)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int32
    for g, w in zip(got[1:], want[1:]):
        assert np.array_equal(g.cpu().numpy(), w), (g.cpu().numpy(), w)
    g, w = got[0].cpu().numpy().astype(np.float64), want[0]
    there = np.isfinite(w)
    assert np.array_equal(g[~there], w[~there])
    assert (np.abs(g[there] - w[there]) <= 5e-6 + 2.0 ** -24 * np.abs(w[there])).all()
    return got


def rows(n, vocab, dtype, seed, pad=0, spread=2.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    held = torch.full((n, vocab + pad), 99.0, dtype=dtype, device="cuda")
    held[:, :vocab] = spread * torch.randn((n, vocab), generator=g, device="cuda")
    return held[:, :vocab]


def begun(requests, beams, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return -5.0 * torch.rand((requests, beams), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("requests,beams,vocab,k,pad", [
    (1, 1, 1, 1, 0), (1, 1, 1, 3, 0), (1, 4, 2, 8, 1), (2, 3, 7, 5, 0), (3, 2, 8, 4, 8), (1, 1, 255, 128, 0), (5, 4, 1000, 8, 1), (1, 4, 32000, 8, 0), (2, 5, 50257, 10, 0),
    (3, 4, 8191, 4, 3), (3, 4, 8192, 4, 0), (3, 4, 8193, 4, 0), (1, 1, 262144, 64, 0), (2, 32, 4099, 64, 5), (1, 64, 3001, 128, 0), (1, 256, 777, 32, 0), (70, 2, 1500, 4, 0),
    (1, 33, 40001, 33, 1), (3, 8, 128000, 16, 0)])
def test_shapes(requests, beams, vocab, k, pad, dtype):
    check(rows(requests * beams, vocab, dtype, vocab + beams, pad), begun(requests, beams, k), k)


def test_a_vocabulary_as_large_as_a_call_takes():
    check(rows(1, 1 << 24, torch.bfloat16, 3), begun(1, 1, 1), 5)


def test_defaults_and_addresses():
    logits, scores = rows(12, 999, torch.float16, 1), begun(3, 4, 1)
    assert all(torch.equal(a, b) for a, b in zip(paged.beam_select(logits, scores), paged.beam_select(logits, scores, 4)))
    wide = rows(12, 1100, torch.float16, 2)
    for first in range(9):  # every address that a row can have
        check(wide[:, first:first + 1000 + first], scores, 6)
    check(wide.as_strided((12, 500), (0, 1)), scores, 6)  # one row for all beams


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits(dtype):
    """Ties go to the lower beam, then to the lower token, however many there are."""
    for vocab in (5, 300, 9000, 50001):
        flat = torch.zeros((8, vocab), dtype=dtype, device="cuda")
        check(flat, torch.zeros((2, 4), device="cuda"), 7)
        check(flat, torch.tensor([[-1.0, 0.0, 0.0, -2.0]] * 2, device="cuda"), 128)
        flat[:, vocab // 2:] = -0.0  # no less than 0
        check(flat, torch.zeros((2, 4), device="cuda"), 7)
    steps = (rows(6, 30000, torch.float32, 5) * 2).round().to(dtype)  # a few dozen values
    check(steps, begun(2, 3, 5), 40)
    same = rows(1, 20000, dtype, 6).expand(6, 20000)
    check(same, torch.zeros((1, 6), device="cuda"), 12)
    check(same.contiguous(), torch.zeros((2, 3), device="cuda"), 12)
    odd = torch.empty((6, 20001), dtype=dtype, device="cuda")  # rows that begin at other addresses
    odd[:, :20000] = same
    check(odd[:, :20000], torch.zeros((1, 6), device="cuda"), 12)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 16, 128])
def test_logits_that_rise_and_fall(dtype, k):
    """The best stand at the end, at the beginning, or all in one thread's share."""
    line = torch.linspace(-6.0, 6.0, 40000, device="cuda").to(dtype)
    together = torch.full((40000,), -3.0, device="cuda", dtype=dtype)
    together[17000:17000 + 600] = torch.linspace(0.0, 5.0, 600, device="cuda").to(dtype)
    for x in (line, line.flip(0), together, -together):
        check(torch.stack((x, x.roll(5), x)), begun(1, 3, 1), k)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_whose_sums_are_nearly_the_same(dtype):
    """Continuations of different beams that 32-bit sums cannot put in order: rows that differ in what weighs least."""
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    base = (2.0 * torch.randn((1, 30011), generator=g, device="cuda")).to(dtype)
    logits = base.repeat(16, 1)
    for i in range(16):  # one logit far below the largest, a different one for each
        logits[i, 100 + i] = -4.0 - 0.25 * ((7 * i) % 16)
    check(logits, torch.zeros((2, 8), device="cuda"), 16)
    check(logits, torch.zeros((1, 16), device="cuda"), 33)
    # scores that make up for the differences to within a few steps of 32 bits
    whole = torch.logsumexp(logits.double(), -1)
    check(logits, (whole - whole[0]).float().view(2, 8), 24)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_the_same_logits_in_another_order(dtype):
    """Their continuations are tied, and go to the lower beam, whatever the order of additions."""
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    for vocab in (2, 3, 10, 1000, 20011):
        base = (2.0 * torch.randn(vocab, generator=g, device="cuda")).to(dtype)
        rows_ = torch.stack([base[torch.randperm(vocab, generator=g, device="cuda")] for _ in range(8)])
        scores, tokens, parents = paged.beam_select(rows_, torch.zeros((1, 8), device="cuda"), 16)
        best_values = rows_.double().sort(dim=-1, descending=True).values[0]  # the same for all rows
        at = 0
        for value in best_values.unique(sorted=True).flip(0).tolist():
            for beam in range(8):
                for token in (rows_[beam].double() == value).nonzero()[:, 0].tolist():
                    if at < min(16, 8 * vocab):
                        assert (tokens[0, at].item(), parents[0, at].item()) == (token, beam), (vocab, at)
                        at += 1
        assert at == min(16, 8 * vocab)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_banned(dtype):
    low = torch.finfo(dtype).min
    for vocab in (40, 20000, 70001):
        logits = rows(8, vocab, dtype, vocab)
        logits[0] = -INF                            # a row without a continuation
        logits[1, 3:] = -INF                        # three are left
        logits[2, :vocab - 1] = -INF                # the last alone
        logits[3] = torch.where(torch.rand(vocab, device="cuda") < 0.97, -INF, logits[3].float()).to(dtype)
        logits[4, ::2] = low                        # masked by the type's lowest value
        logits[5] = low
        logits[6, 1::2] = float("nan")              # weighs nothing
        logits[7] = float("nan")
        check(logits, begun(1, 8, 1), 24)
        check(logits, begun(4, 2, 2), 9)
        check(logits, begun(8, 1, 3), 5)
        check(logits.roll(3, 1), begun(2, 4, 3), 128)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_logits(dtype):
    logits = rows(4, 30000, dtype, 1)
    logits[0, 20000] = INF
    logits[1, [5, 29999, 11]] = INF
    logits[1, 12] = float("nan")
    logits[2] = INF
    check(logits, begun(1, 4, 1), 8)
    check(logits, begun(4, 1, 1), 8)


def test_beams_that_have_not_begun():
    logits = rows(12, 5000, torch.bfloat16, 1)
    logits[[1, 2, 3]] = float("nan")
    scores = torch.tensor([[0.0, -INF, -INF, -INF], [-INF, float("nan"), -3.0, INF], [-INF] * 4], device="cuda")
    got = check(logits, scores, 10)
    assert (got[1][2] == -1).all() and (got[2][2] == -1).all() and (got[0][2] == -INF).all()
    assert set(got[2][0].tolist()) == {0} and set(got[2][1].tolist()) == {6}


def test_large_and_small_logits():
    for offset in (1e4, -3e4, 1e30, -1e30):
        check(rows(4, 9000, torch.float32, 1) + offset, begun(1, 4, 1), 8)
    check(rows(4, 9000, torch.float32, 1) * 1e-30, begun(1, 4, 1), 8)
    check(rows(4, 9000, torch.float32, 1) * 1e36, begun(1, 4, 1), 8)
    check(rows(4, 9000, torch.float32, 2), begun(1, 4, 1) * 1e6, 8)


def test_no_requests():
    got = paged.beam_select(torch.empty((0, 100), dtype=torch.float16, device="cuda"), torch.empty((0, 4), device="cuda"))
    assert all(t.shape == (0, 4) for t in got)


def test_the_same_every_time_and_in_a_graph():
    logits, scores = rows(64, 33001, torch.bfloat16, 1), begun(8, 8, 1)
    first = check(logits, scores, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0], stream=side):
        one = paged.beam_select(logits, scores, 16)
    with torch.cuda.graph(graphs[1], stream=side):  # with a workspace of its own
        two = paged.beam_select(logits, scores, 16)
    for n in range(20):
        graphs[n % 2].replay()
        now = one if n % 2 == 0 else two
        assert all(torch.equal(a, b) for a, b in zip(now, first))
    logits.copy_(rows(64, 33001, torch.bfloat16, 2))
    with torch.cuda.stream(side):
        graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    again = check(logits, scores, 16)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(again, one, two))
