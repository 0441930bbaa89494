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


def put(b, request, key, head, column, value):
    b.v[b.table[request].long()[key // 16], key % 16, head, column] = value


def agrees(b, **how):
    """Numbers within the tolerance, and infinities and values that are no numbers where the formula has them."""
    out, _ = b.call(**how)
    want, _, tol = attention(b.q, b.k, b.v, b.table, b.lens, b.scale, **how)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isposinf(), want.isposinf()) and torch.equal(out.isneginf(), want.isneginf())
    fine = want.isfinite()
    assert bool(((out.double() - want).abs() <= tol)[fine].all())
    return want


def milliseconds(call):
    """The least of five, by events, with the call captured, so that the host's part is not in it."""
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    times = []
    for _ in range(5):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        graph.replay()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    return min(times)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
def test_a_value_that_is_not_finite_and_that_all_see_costs_nothing(dtype):
    """An infinite value of a prompt's first token reaches every row by right: rows are not done again one by one, key by key, which takes
    hundreds of times as long.  Neither are they where all values are no numbers.  (Bounds with room: three times, and 0.2 ms.)"""
    b = Batch([(2000, 2000)], 8, 8, 128, 16, dtype)
    usual = milliseconds(b.call)
    put(b, 0, 0, 3, 100, math.inf)
    want = agrees(b)
    assert bool(want[:, 3, 100].isposinf().all()) and int(want.isinf().sum()) == 2000
    assert milliseconds(b.call) <= 3 * usual + 0.2
    b.v.fill_(math.nan)
    out, lse = b.call()
    assert bool(out.isnan().all()) and bool(lse.isfinite().all())
    assert milliseconds(b.call) <= 3 * usual + 0.2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("lens,q_heads,heads,head,how", [
    ([(200, 9000)], 2, 2, 128, {}), ([(300, 4000), (40, 700)], 4, 2, 64, {}), ([(300, 1100)], 2, 2, 64, dict(window=150)),
    ([(120, 1500)], 2, 1, 128, dict(window=300)), ([(150, 700)], 4, 4, 80, dict(window=64, causal=False)), ([(14, 600), (5, 5)], 2, 2, 128, dict(window=200)),
    ([(260, 100)], 2, 2, 64, {})], ids=ids)
def test_values_that_are_not_finite_anywhere(lens, q_heads, heads, head, how, dtype):
    """Infinities and values that are no numbers at keys that all rows of a tile see, some or none; in tiles that are divided and in whole
    ones, in blocks at the borders of what rows see."""
    b = Batch(lens, q_heads, heads, head, 16, dtype, seed=5)
    g = torch.Generator()
    g.manual_seed(len(lens) + lens[0][0])
    for request, (n, kv) in enumerate(lens):
        places = [0, kv - 1, kv - 2] + torch.randint(0, kv, (4,), generator=g).tolist() + torch.randint(max(0, kv - n), kv, (6,), generator=g).tolist()
        for i, key in enumerate(places):
            column = int(torch.randint(0, head, (1,), generator=g))
            put(b, request, key, i % heads, column, (math.inf, -math.inf, math.nan)[i % 3])
    want = agrees(b, **how)
    assert int((~want.isfinite()).sum()) > 0


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_new_values_that_are_all_not_finite(value):
    """Every row is done again, or none, and each sees what it should."""
    b = Batch([(140, 900), (300, 300)], 2, 2, 64, 16, torch.bfloat16)
    for request, (n, kv) in enumerate([(140, 900), (300, 300)]):
        j = torch.arange(kv - n, kv, device="cuda")
        b.v[b.table[request].long()[j // 16], j % 16, 1] = value
    want = agrees(b)
    assert bool(want[:, 0].isfinite().all()) and not want[:, 1].isfinite().any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("n,requests", [(1, 600), (20, 160)])
def test_many_small_weights_beside_a_large_one(n, requests, dtype):
    """One key with a score of 17.375 and values 0 over a million with score 0 and values 1: each of these has 2^-25.07 of its weight, below half the
    smallest fp16 number, and all together S = 3 %, so the result is S / (1 + S).  (Of more requests than there are blocks, so that blocks
    have whole requests: parts without the large weight are relative to the small ones.)

    Tolerance, as a share of the result: its rounding by half a step; that of a weight, by half a step in the rows' kernel; in the other, where
    2^-18.07 is what fp16 has of it, by 2^-25, 0.8 %.  32-bit sums: up to 2^16 steps of 16 products, each off by 2^-23 of half the sum on average
    (products may cut off): 0.4 %; and in the sum of weights a thread adds one at a time to the large one, for a quarter of a quarter of the
    keys, and may lose all of these: S / 16, 0.2 %; exponents of 25 in 32 bits 2^-20.

    With values of 1 at that key too the result is 1.  A 32-bit sum that has reached 1 may lose summands below 2^-24 of it whole, and these
    are: the small weights that are summed with the large one, S / 4 of single rows (by one of four warps), S / 2 of chunks (by one of two groups)."""
    from cachegen_b200 import paged
    kv, D, page = 2 ** 20, 8, 64
    k, v = torch.zeros((kv // page, page, 1, D), dtype=dtype, device="cuda"), torch.ones((kv // page, page, 1, D), dtype=dtype, device="cuda")
    q = torch.zeros((n * requests, 1, D), dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    table = torch.arange(kv // page, dtype=torch.int32, device="cuda").expand(requests, -1)
    lens = torch.full((requests,), kv, dtype=torch.int32, device="cuda")
    starts = torch.arange(0, n * requests + 1, n, dtype=torch.int32, device="cuda")
    score = 17.375  # a bf16 number
    half = torch.finfo(dtype).eps / 2
    for main in (0, 500_000, kv - n):
        k.zero_(), v.fill_(1)
        k[main // page, main % page, 0, 0] = score
        v[main // page, main % page] = 0
        out, lse = paged.paged_attention(q, k, v, table, lens, starts, scale=1.0, max_q=n, return_lse=True)
        small = torch.arange(kv - n, kv, device="cuda").double().repeat(requests)[:, None] * math.exp(-score)
        want = (small / (1 + small))[..., None]
        off = ((out.double() - want).abs() / want).max().item()
        beside, _ = paged.paged_attention(q, k, torch.ones_like(v), table, lens, starts, scale=1.0, max_q=n, return_lse=True)
        assert bool(((beside.double() - 1).abs() <= half + 0.001 + (small * (1 / 16 + (1 / 4 if n == 1 else 1 / 2)))[..., None]).all())
        assert off <= 2 * half + 0.004 + 0.002 + (0.008 if n > 1 and dtype == torch.float16 else 0), off
        # the sum of weights as above, and the logarithm's rounding, a step of 17 2^-19
        assert bool(((lse.double() - score - torch.log1p(small)).abs() <= small / 16 + 2.0 ** -18).all())
    paged.check_status()


def test_rows_beside_each_other_are_taken_and_overlapping_ones_refused(monkeypatch):
    """Queries, keys and values of one array, rotated in place, by the native call too; what a block would write while another reads it is
    refused by both paths."""
    from cachegen_b200 import _lib, paged
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    qkv = torch.randn((9, 8, 64), generator=g, device="cuda").half()
    pages = torch.zeros((3, 4, 2, 2, 64), dtype=torch.float16, device="cuda")
    rotary, slots, at = paged.Rotary(64), torch.arange(9, device="cuda"), torch.arange(5, 14, device="cuda")
    k_pages, v_pages = pages[:, :, 0], pages[:, :, 1]
    want = [paged.apply_rotary(qkv[:, :4], at, rotary), paged.apply_rotary(qkv[:, 4:6], at, rotary), qkv[:, 6:].clone()]
    taken, entry = [], _lib.native_calls().append
    monkeypatch.setattr(_lib.native_calls(), "append", lambda *a: taken.append(entry(*a)) or taken[-1])
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    assert paged.append_paged(k, v, k_pages, v_pages, slots, rotary=rotary, positions=at, q=q, q_out=q) is q and taken[0] is q
    assert torch.equal(q, want[0]) and torch.equal(pages.view(12, 2, 2, 64)[:9, 0], want[1]) and torch.equal(pages.view(12, 2, 2, 64)[:9, 1], want[2])
    kv = torch.zeros((9, 2, 2, 64), dtype=torch.float16, device="cuda")
    paged.gather_paged(k_pages, v_pages, slots, k=kv[:, 0], v=kv[:, 1])
    assert torch.equal(kv, pages.view(12, 2, 2, 64)[:9])
    some = k.contiguous()
    for refused in (dict(q=some, q_out=k), dict(q=some, q_out=v), dict(q=some, q_out=qkv[:, 5:7]), dict(q=some, q_out=pages[0, 0, 0][None].expand(9, -1, -1)),
                    dict(q=k_pages.reshape(12, 2, 64)[:9], q_out=pages.view(24, 2, 64)[:9]), dict(q=pages.view(24, 2, 64)[1:10])):
        with pytest.raises(RuntimeError):
            paged.append_paged(k, v, k_pages, v_pages, slots, **refused)
    with pytest.raises(RuntimeError):
        paged.append_paged(k, v, pages.view(24, 1, 2, 64)[:12], pages.view(24, 1, 2, 64)[6:18], slots)
    with pytest.raises(RuntimeError):
        paged.gather_paged(k_pages, v_pages, slots, k=some, v=some)
    paged.check_status()


def test_what_is_written_to_has_a_new_version(monkeypatch):
    """Of the native calls and of the Python path: a backward pass that kept such a tensor refuses it."""
    from cachegen_b200 import _lib, _plain_calls, paged
    rotary, at = paged.Rotary(64), torch.arange(6, device="cuda")
    table, lens = torch.zeros((6, 1), dtype=torch.int32, device="cuda"), torch.ones(6, dtype=torch.int32, device="cuda")

    def rows(*shape):
        return torch.zeros(shape, dtype=torch.float16, device="cuda")
    calls = (lambda x, o: paged.apply_rotary(x, at, rotary, out=x), lambda x, o: paged.append_paged(o, o, x.view(6, 1, 2, 64), rows(6, 1, 2, 64), at),
             lambda x, o: paged.append_paged(o, o, rows(6, 1, 2, 64), x.view(6, 1, 2, 64), at), lambda x, o: paged.append_paged(
                 o, o, rows(6, 1, 2, 64), rows(6, 1, 2, 64), at, q=o, q_out=x),
             lambda x, o: paged.gather_paged(rows(6, 1, 2, 64), rows(6, 1, 2, 64), at, k=x), lambda x, o: paged.gather_paged(
                 rows(6, 1, 2, 64), rows(6, 1, 2, 64), at, v=x),
             lambda x, o: paged.paged_attention(o, rows(1, 16, 2, 64), rows(1, 16, 2, 64), table, lens, out=x))
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "_calls", _plain_calls)
        for call in calls:
            x, weight = rows(6, 2, 64), rows(6, 2, 64).requires_grad_()
            y = (weight * x).sum()
            call(x, rows(6, 2, 64))
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
            with torch.inference_mode():
                call(rows(6, 2, 64), rows(6, 2, 64))
                of_inference = rows(6, 2, 64)
            call(of_inference, rows(6, 2, 64))
    paged.check_status()


@pytest.mark.parametrize("native", [True, False])
def test_a_rotary_may_be_dropped_while_another_stream_uses_it(native, monkeypatch):
    """Its memory is not handed out again before that stream is done.  (Nothing is written to what is handed out.)"""
    from cachegen_b200 import _lib, _plain_calls, paged
    if not native:
        monkeypatch.setattr(_lib, "_calls", _plain_calls)
    x, at = torch.ones((4, 2, 128), dtype=torch.float16, device="cuda"), torch.arange(4, device="cuda")
    pages = torch.zeros((2, 1, 16, 2, 128), dtype=torch.float16, device="cuda")
    calls = (lambda r: paged.apply_rotary(x, at, r), lambda r: paged.append_paged(x, x, pages[0], pages[1], at, rotary=r, positions=at),
             lambda r: paged.gather_paged(pages[0], pages[1], at, rotary=r, positions=at))
    side = torch.cuda.Stream()
    for call in calls:
        call(paged.Rotary(128))
        torch.cuda.synchronize()
        rotary = paged.Rotary(128)
        address = rotary.turns(x.device).data_ptr()
        with torch.cuda.stream(side):
            torch.cuda._sleep(400_000_000)
            call(rotary)
        del rotary
        handed_out = [torch.empty(64, dtype=torch.int64, device="cuda") for _ in range(100)]
        assert not side.query()  # it waits still
        assert address not in [t.data_ptr() for t in handed_out]
        torch.cuda.synchronize()
    paged.check_status()


def test_a_rotary_can_be_copied():
    import copy
    import pickle
    from cachegen_b200 import paged
    x, at = torch.randn((4, 2, 64), device="cuda").half(), torch.arange(4, device="cuda")
    r = paged.Rotary(64, rotary_dims=32, scaling=("linear", 2.0))
    want = paged.apply_rotary(x, at, r)
    for other in (copy.copy(r), copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert other.frequencies == r.frequencies and torch.equal(paged.apply_rotary(x, at, other), want)
        assert other.turns(x.device) is not r.turns(x.device)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("n", [1, 20])
def test_the_longest_request(n, dtype):
    """2^30 keys, of two pages that are named again and again, one with values of 1 and one of 3.  Scores are 0: sums of 1 and 3 are exact in 32 bits
    up to 2^24, a block's share has fewer, and joined they are powers of two or three quarters of one."""
    from cachegen_b200 import paged
    kv, page = 2 ** 30, 128
    k, v = torch.zeros((2, page, 1, 8), dtype=dtype, device="cuda"), torch.ones((2, page, 1, 8), dtype=dtype, device="cuda")
    v[1] = 3
    table = torch.zeros((1, kv // page), dtype=torch.int32, device="cuda")
    table[0, 1::2] = 1
    q = torch.ones((n, 1, 8), dtype=dtype, device="cuda")
    lens, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([kv], [0, n]))
    for window in (0, 2 ** 29, 2 ** 30):
        out, lse = paged.paged_attention(q, k, v, table, lens, starts, return_lse=True, window=window, max_q=n)
        paged.check_status()
        assert bool(((out.double() - 2).abs() <= 2 * torch.finfo(dtype).eps / 2 + 2.0 ** -10).all())
        assert bool(((lse.double() - math.log(window or kv)).abs() <= 2.0 ** -18).all())  # (n keys more or less are nothing beside 2^29)
