"""Attention over a paged cache against softmax in 64 bits."""
import math

import pytest
import torch

from paged_ref import attention

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


class Batch:
    """Requests (new tokens, keys) with their pages in random order, NaN wherever nothing may be read."""

    def __init__(self, lens, q_heads, heads, head, page, dtype, transposed=False, seed=0, extra_rows=0, spread=1.0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        need = [(kv + page - 1) // page for _, kv in lens]
        pool = sum(need) + 2
        order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), max(need) + 1), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
        shape = (pool, heads, page, head) if transposed else (pool, page, heads, head)
        self.k, self.v = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2))
        if transposed:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        at, first, self.lens, starts = 0, 0, [], [0]
        for b, ((n, kv), m) in enumerate(zip(lens, need)):
            pages = order[at:at + m]
            self.table[b, :m] = pages
            j = torch.arange(kv, device="cuda")
            for t in (self.k, self.v):
                t[pages.long()[j // page], j % page] = (spread * torch.randn((kv, heads, head), generator=g, device="cuda")).to(dtype)
            self.lens.append((first, n, kv))
            at, first = at + m, first + n
            starts.append(first)
        self.rows = first
        self.q = (spread * torch.randn((first + extra_rows, q_heads, head), generator=g, device="cuda")).to(dtype)
        self.kv_lens = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
        self.q_starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.scale = 1.0 / math.sqrt(head)

    def call(self, **more):
        from cachegen_b200 import paged
        return paged.paged_attention(self.q, self.k, self.v, self.table, self.kv_lens, self.q_starts, return_lse=True, **more)

    def check(self, got, lse, scale=None, **how):
        from cachegen_b200 import paged
        paged.check_status()
        want, want_lse, tol = attention(self.q, self.k, self.v, self.table, self.lens, self.scale if scale is None else scale, **how)
        R = self.rows
        assert torch.equal(got[:R].isnan(), want[:R].isnan())
        off = (got[:R].double() - want[:R]).abs()
        assert bool((off <= tol[:R]).all()), f"off by {off.nan_to_num().max().item()}, {(off / tol[:R].clamp(min=1e-30)).nan_to_num().max().item()} times the tolerance"
        empty = want_lse[:R] == -math.inf
        assert torch.equal(empty, lse[:R] == -math.inf)
        # scores as above, the sum of weights by 2^-22 a weight (its exponential), and the logarithm
        D = self.q.shape[2]
        reach = (self.q.double().abs().sum(-1)[:R] * self.k.double().nan_to_num().abs().max() * abs(self.scale if scale is None else scale))
        assert bool(((lse[:R].double() - want_lse[:R]).abs()[~empty] <= ((D + 8) * 2.0 ** -23 * reach + 2.0 ** -19 * (1 + want_lse[:R].abs()))[~empty]).all())


def ids(v):
    return str(v).replace(" ", "").replace("torch.", "")


STEPS = [  # lens, q heads, heads, head, page
    ([(1, 1)], 4, 1, 128, 16), ([(1, 61)], 32, 8, 128, 16), ([(1, 64)], 8, 8, 64, 16), ([(1, 65)], 8, 8, 64, 16), ([(1, 4097)], 32, 8, 128, 64),
    ([(1, 0), (1, 5), (1, 300), (1, 1)], 8, 2, 128, 16), ([(1, 1000), (1, 20), (1, 517)], 16, 1, 128, 1), ([(1, 129), (1, 2)], 7, 1, 80, 24),
    ([(1, 200)], 12, 12, 96, 7), ([(1, 90), (1, 91)], 2, 1, 8, 16), ([(1, 333)], 6, 3, 40, 128), ([(1, 77)], 3, 1, 72, 16),
    ([(1, 257)] * 40, 4, 4, 64, 16), ([(2, 300), (4, 4), (1, 9), (3, 70)], 8, 2, 128, 16), ([(16, 50), (5, 1000)], 2, 2, 128, 16),
    ([(1, 3000)], 16, 16, 128, 16)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lens,q_heads,heads,head,page", STEPS, ids=ids)
def test_steps(lens, q_heads, heads, head, page, dtype):
    b = Batch(lens, q_heads, heads, head, page, dtype, transposed=len(lens) == 3)
    b.check(*b.call(max_q=max(n for n, _ in lens)))


def test_steps_without_starts():
    from cachegen_b200 import paged
    b = Batch([(1, 100), (1, 3), (1, 0)], 8, 2, 128, 16, torch.bfloat16)
    b.q_starts = None
    b.check(*b.call())
    assert paged.paged_attention(b.q, b.k, b.v, b.table, b.kv_lens).shape == b.q.shape


CHUNKS = [  # lens, q heads, heads, head, page
    ([(17, 17)], 1, 1, 128, 16), ([(64, 64)], 8, 8, 128, 16), ([(100, 1000)], 8, 2, 128, 16), ([(256, 300)], 4, 4, 64, 128),
    ([(33, 4000), (1, 700), (0, 50), (129, 129)], 8, 2, 128, 16), ([(300, 300), (7, 2000)], 7, 1, 80, 24), ([(70, 90)], 3, 3, 96, 5),
    ([(20, 10), (40, 40), (5, 0)], 4, 1, 64, 16), ([(513, 513)], 2, 1, 128, 64), ([(18, 200)] * 30, 4, 4, 128, 16), ([(50, 50)], 6, 2, 24, 1),
    ([(1, 900), (2, 800), (60, 60)], 64, 1, 128, 16), ([(700, 1500)], 2, 2, 128, 16)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lens,q_heads,heads,head,page", CHUNKS, ids=ids)
def test_chunks(lens, q_heads, heads, head, page, dtype):
    b = Batch(lens, q_heads, heads, head, page, dtype, transposed=len(lens) == 2)
    b.check(*b.call())


@pytest.mark.parametrize("lens,heads", [([(1, 500), (1, 30)], 8), ([(100, 700), (300, 300)], 2), ([(9, 400)], 4)], ids=ids)
@pytest.mark.parametrize("window", [1, 5, 64, 250, 100000])
@pytest.mark.parametrize("causal", [True, False])
def test_windows_and_no_causality(lens, heads, window, causal):
    b = Batch(lens, 8, heads, 64, 16, torch.float16)
    b.check(*b.call(window=window, causal=causal), window=window, causal=causal)


@pytest.mark.parametrize("lens", [[(1, 300)], [(40, 300)], [(300, 300)]], ids=ids)
def test_not_causal(lens):
    b = Batch(lens, 4, 2, 128, 16, torch.bfloat16)
    b.check(*b.call(causal=False), causal=False)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.5, 4.0])
@pytest.mark.parametrize("lens", [[(1, 300)], [(150, 400)]], ids=ids)
def test_scales(lens, scale):
    """Large scores: one key has nearly all the weight, and the running maximum rises far."""
    b = Batch(lens, 4, 2, 128, 16, torch.bfloat16)
    b.check(*b.call(scale=scale), scale=scale)


@pytest.mark.parametrize("lens", [[(1, 500)], [(140, 600)], [(3, 200)]], ids=ids)
def test_a_maximum_that_keeps_rising(lens):
    """Keys in rising order of their scores, so that every block has a new maximum, and in falling order."""
    for order in (1, -1):
        b = Batch(lens, 4, 2, 64, 16, torch.float16)
        kv = lens[0][1]
        b.q.fill_(1.0)
        ramp = torch.linspace(-40, 40, kv, device="cuda")[:, None, None].expand(kv, 2, 64) / 8
        j = torch.arange(kv, device="cuda")
        b.k[b.table[0].long()[j // 16], j % 16] = (ramp if order > 0 else ramp.flip(0)).half()
        b.check(*b.call())


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens,q_heads", [([(6, 100)], 2), ([(40, 300)], 2), ([(300, 300)], 8), ([(1, 50), (4, 20)], 2)], ids=ids)
def test_values_of_hidden_keys_stay_out(lens, q_heads, value):
    """A new token's key and value are not finite: the tokens before it do not see them, those behind it do."""
    for bad_k, bad_v in ((True, True), (False, True)):
        b = Batch(lens, q_heads, 2, 64, 16, torch.bfloat16)
        n, kv = lens[-1]
        j = kv - n // 2 - 1
        page = b.table[len(lens) - 1].long()[j // 16]
        b.v[page, j % 16, 1, 3] = value
        if bad_k:
            b.k[page, j % 16, 1, 5] = math.nan
        out, lse = b.call()
        want, _, tol = attention(b.q, b.k, b.v, b.table, b.lens, b.scale)
        assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf())
        fine = want.isfinite()
        assert bool(((out.double() - want).abs() <= tol)[fine].all()) and int((~fine).sum()) > 0


def test_rows_of_no_request_and_strided_rows():
    b = Batch([(3, 40), (2, 9)], 8, 2, 64, 16, torch.float16, extra_rows=4)
    wide = torch.full((9, 8, 3 * 64), math.nan, dtype=torch.float16, device="cuda")
    wide[:, :, 64:128] = b.q
    b.q = wide[:, :, 64:128]
    out = torch.full((9, 8, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    got, lse = b.call(out=out[:, :, 1])
    b.check(got, lse)
    assert bool((out[:, :, 0] == 7).all()) and bool((out[5:] == 7).all())


def test_nothing_to_do():
    from cachegen_b200 import paged
    b = Batch([(1, 10)], 4, 2, 64, 16, torch.float16)
    none = b.q[:0]
    assert paged.paged_attention(none, b.k, b.v, b.table[:0], b.kv_lens[:0]).shape == (0, 4, 64)
    starts = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.full_like(b.q, 3.0)
    paged.paged_attention(b.q, b.k, b.v, b.table, b.kv_lens, starts, out=out)  # a request without new tokens
    paged.check_status()
    assert bool((out == 3).all())
    zero = torch.zeros_like(b.kv_lens)
    assert not paged.paged_attention(b.q, b.k, b.v, b.table[:, :0], zero).any()  # no page at all


def test_what_does_not_fit_is_cut_and_reported():
    from cachegen_b200 import paged
    for lens in ([(1, 40), (1, 40)], [(30, 40), (20, 40)]):
        b = Batch(lens, 4, 2, 64, 16, torch.float16)
        b.table = b.table[:, :3].contiguous()
        good = b.call(max_q=lens[0][0])
        kv = b.kv_lens.clone()
        for change, spared in ((lambda: b.kv_lens.copy_(torch.tensor([40, 49], dtype=torch.int32)), 0),
                               (lambda: b.kv_lens.copy_(torch.tensor([-1, 40], dtype=torch.int32)), 1),
                               (lambda: b.table[0].fill_(-5), 1), (lambda: b.table[0].fill_(10 ** 9), 1),
                               (lambda: b.q_starts.copy_(torch.tensor([0, lens[0][0], 10 ** 6], dtype=torch.int32)), 0)):
            table, starts = b.table.clone(), b.q_starts.clone()
            change()
            out, _ = b.call(max_q=lens[0][0])
            with pytest.raises(RuntimeError, match="paged cache"):
                paged.check_status()
            first, n, _ = b.lens[spared]
            assert torch.equal(out[first:first + n], good[0][first:first + n])
            b.table.copy_(table), b.q_starts.copy_(starts), b.kv_lens.copy_(kv)
        b.check(*b.call())


def test_offsets_beyond_32_bits():
    from cachegen_b200 import paged
    store = torch.zeros(2 ** 31 + 2 ** 21, dtype=torch.float16, device="cuda")
    for n in (1, 40):
        b = Batch([(n, 40)], 4, 2, 64, 16, torch.float16)
        far = [store.as_strided((3, 16, 2, 64), (2 ** 30, 128, 64, 1), at) for at in (0, 2 ** 20)]
        for t, s in zip(far, (b.k, b.v)):
            t.copy_(s[b.table[0, :3].long()])
        b.k, b.v = far
        b.table[0, :3] = torch.tensor([0, 1, 2], dtype=torch.int32)
        b.check(*b.call())


def test_the_same_result_every_time_and_in_any_company():
    """A request's result does not depend on the order of the blocks that work on it: two calls give the same bits."""
    for lens in ([(1, 5000), (1, 40)], [(60, 3000), (200, 900)]):
        b = Batch(lens, 8, 2, 128, 16, torch.bfloat16)
        first = b.call()
        for _ in range(5):
            again = b.call()
            assert all(torch.equal(x, y) for x, y in zip(first, again))


@pytest.mark.parametrize("n", [1, 50])
def test_graphs_follow_the_lengths_and_do_not_share(n):
    """Two captured graphs, replayed in turn and at the same time; lengths change between replays."""
    batches = [Batch([(n, 3000), (n, 700)], 8, 2, 128, 16, torch.bfloat16, seed=s) for s in (1, 2)]
    graphs, results = [], []
    for b in batches:
        b.call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(b.call(max_q=n))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for lens in ([3000, 700], [n, 64], [1024, 699]):
        for b in batches:
            b.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            b.lens = [(first, m, kv) for (first, m, _), kv in zip(b.lens, lens)]
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for b, r in zip(batches, results):
            b.check(*r)


def test_many_requests():
    from cachegen_b200 import _lib
    lens = [(1, 1 + i % 90) for i in range(_lib.CG_MAX_REQUESTS)]
    b = Batch(lens, 2, 1, 16, 16, torch.float16)
    out, lse = b.call(max_q=1)
    for i in (0, 1, 77, 2048, 4095):
        n, kv = lens[i]
        j = torch.arange(kv, device="cuda")
        rows = b.table[i].long()[j // 16], j % 16
        k, v = b.k[rows][:, 0].double(), b.v[rows][:, 0].double()
        w = torch.softmax(b.q[i].double() @ k.T * b.scale, -1)
        # weights of 16 bits and the result's rounding, as in paged_ref.attention
        assert bool(((out[i].double() - w @ v).abs() <= 2.0 ** -11 * ((w @ v).abs() + 1.1 * (w @ v.abs())) + 2.0 ** -15).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("page", [8, 16, 32, 96, 128])
@pytest.mark.parametrize("head", [8, 40, 64, 72, 128])
def test_chunks_of_every_box(head, page, dtype):
    """Pages that are read a box of tokens at a time, heads that fill a box and that do not; lengths that end inside a box; with
    heads outside and inside of tokens."""
    for transposed in (False, True):
        b = Batch([(40, 40), (65, 333), (30, 200)], 4, 2, head, page, dtype, transposed=transposed, seed=head + page)
        b.check(*b.call())
    b.check(*b.call(window=77), window=77)


def test_a_hint_that_is_too_small_costs_time_only():
    b = Batch([(300, 900), (1, 50)], 4, 2, 64, 16, torch.float16)
    b.check(*b.call(max_q=1))


@pytest.mark.parametrize("n", [1, 40])
def test_one_key_value_head_of_many_and_strides_of_one_page(n):
    """Pages and heads that are views of a larger cache: every stride differs from the contiguous one."""
    big = torch.full((7, 16, 6, 3 * 64), math.nan, dtype=torch.float16, device="cuda")
    b = Batch([(n, 60)], 4, 2, 64, 16, torch.float16)
    pages = b.table[0, :4].long()
    k, v = big[::2, :, ::3, 64:128], big[::2, :, 1::3, 128:]  # every second page, every third head, the middle and last 64 values
    k.copy_(b.k[pages]), v.copy_(b.v[pages])
    b.k, b.v, b.table = k, v, torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device="cuda")
    b.check(*b.call())


def test_a_capture_in_front_of_any_call(monkeypatch):
    """The status word is not made of a graph's memory."""
    from cachegen_b200 import paged, torchac_cuda
    b = Batch([(1, 70)], 4, 2, 64, 16, torch.float16)
    b.call()
    words = {}
    monkeypatch.setattr(paged, "_status", words)
    monkeypatch.setattr(torchac_cuda, "_status", words)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.call()
    assert not words
    graph.replay()
    b.check(*out)


@pytest.mark.parametrize("page", [1, 5, 16, 24, 64])
@pytest.mark.parametrize("head", [64, 128])
def test_few_rows_over_many_keys(head, page):
    """Between one row and 128 a key/value head: from one block of keys to dozens, whole and divided, of pages of every kind."""
    b = Batch([(5, 1), (20, 100), (9, 129), (30, 300), (17, 1500), (32, 5000), (25, 700)], 8, 2, head, page, torch.bfloat16, seed=page)
    b.check(*b.call())
    b.check(*b.call(window=333), window=333)


def test_few_rows_of_many_requests_at_once():
    """More tiles than blocks of a GPU, so that one block has several, of few rows and of many."""
    lens = [(3 + 5 * (i % 11), 40 + 97 * (i % 13)) for i in range(60)]
    lens = [(n, max(n, kv)) for n, kv in lens]
    b = Batch(lens, 16, 4, 64, 16, torch.float16)
    b.check(*b.call())


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_values_of_hidden_keys_stay_out_of_few_rows_over_many_keys(value):
    b = Batch([(30, 700)], 4, 2, 64, 16, torch.float16)
    j = 690
    b.v[b.table[0].long()[j // 16], j % 16, 1, 3] = value
    out, _ = b.call()
    want, _, tol = attention(b.q, b.k, b.v, b.table, b.lens, b.scale)
    fine = want.isfinite()
    assert torch.equal(out.isfinite(), fine) and int((~fine).sum()) == 10 * 2 and bool(((out.double() - want).abs() <= tol)[fine].all())


def test_arguments_of_kindred_types():
    """Numbers for truth values, whole numbers and arrays' elements for floats: the same call."""
    import numpy as np
    b = Batch([(20, 50), (3, 9)], 4, 2, 64, 16, torch.float16)
    for causal in (True, False):
        want = b.call(causal=causal, scale=1.0, window=16)
        for kind in (int, np.bool_):
            got = b.call(causal=kind(causal), scale=1, window=16)
            assert all(torch.equal(x, y) for x, y in zip(want, got))
        assert all(torch.equal(x, y) for x, y in zip(want, b.call(causal=causal, scale=np.float64(1.0), window=16)))
