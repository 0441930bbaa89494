"""Pages that rows share: forked, extended, given back and moved, against the same steps one by one on the host.  All of it is whole numbers
and copies: equality, and what no call names stays bit for bit."""
import random

import pytest
import torch

from cachegen_b200 import paged
from pages_ref import Cache, need

pytestmark = pytest.mark.gpu


def numbers(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def bits(t):
    return t.view(torch.int16)


def pool(layers, pages, page, heads, head, dtype=torch.float16, fmt="vllm", seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    shape = (layers, 2, pages) + ((heads, page) if fmt == "huggingface" else (page, heads)) + (head,)
    cache = torch.randint(-2 ** 15, 2 ** 15, shape, generator=g, device="cuda", dtype=torch.int16).view(dtype)
    return cache, paged.split_pages(cache, fmt)


def moved(t, moves):
    """t [..., pages, page, heads, head] with the first n tokens of page a copied to page b, for (a, b, n)"""
    out = t.clone()
    for a, b, n in moves:
        bits(out)[..., b, :n, :, :] = bits(t)[..., a, :n, :, :]
    return out


def layout(rng, rows, pages, page, width, share=0.5, longest=None):
    """A cache of rows that share their first pages with the row in front, and the GPU's copy of it."""
    order = rng.sample(range(pages), pages)
    table, lens = [], []
    for r in range(rows):
        n = rng.randint(0, (longest or width * page))
        row = [order.pop() if order else -1 for _ in range(need(n, page))]
        if -1 in row:
            n, row = 0, []
        if r and rng.random() < share:
            common = min(lens[-1] // page, n // page, rng.randint(0, width))
            order += row[:common]
            row[:common] = table[-1][:common]
        table.append(row + [-1] * (width - len(row)))
        lens.append(n)
    cache = Cache(pages, page, table, lens)
    return cache, numbers(table).view(rows, width), numbers(lens).view(rows), numbers(cache.refs)


SHAPES = [  # rows, pages, page, width
    (1, 1, 1, 1), (1, 9, 16, 3), (4, 50, 16, 8), (7, 40, 1, 5), (33, 500, 24, 17), (64, 4099, 8, 63), (300, 9000, 16, 40), (5, 20000, 64, 1500)]


@pytest.mark.parametrize("rows,pages,page,width", SHAPES)
@pytest.mark.parametrize("release", [True, False])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_fork(rows, pages, page, width, release, wide):
    rng = random.Random(rows * 1000 + pages + release)
    paged.check_status()
    for new in (rows, 1, 2 * rows + 1):
        cache, table, lens, refs = layout(rng, rows, pages, page, width, longest=max(1, min(width * page, pages * page // (2 * rows))))
        parents = [rng.choice([-1] + list(range(rows)) * 4) for _ in range(new)]
        if len(cache.free()) < new:
            parents = parents[:len(cache.free())]
        before = table.clone(), lens.clone()
        got, got_lens, moves = paged.fork_pages(table, lens, numbers(parents, wide), refs, page_size=page, release=release)
        want, want_lens, copies, lost = cache.fork(parents, release)
        assert not lost
        assert got.tolist() == want and got_lens.tolist() == want_lens and refs.tolist() == cache.refs
        assert moves.tolist() == [[c[i] for c in copies] + [-1] * (len(parents) - len(copies)) for i in range(3)]
        assert torch.equal(table, before[0]) and torch.equal(lens, before[1])
    paged.check_status()


@pytest.mark.parametrize("layers,page,heads,head", [(1, 16, 8, 128), (3, 16, 2, 64), (2, 5, 3, 40), (2, 8, 1, 7), (0, 64, 2, 80), (1, 1, 1, 8)])
@pytest.mark.parametrize("dtype,fmt", [(torch.float16, "vllm"), (torch.bfloat16, "huggingface")])
def test_fork_copies_the_last_pages(layers, page, heads, head, dtype, fmt):
    rng = random.Random(page + head)
    cache, table, lens, refs = layout(rng, 6, 60, page, 4)
    held, (k, v) = pool(max(1, layers), 60, page, heads, head, dtype, fmt)
    if not layers:
        k, v = k[0], v[0]
    parents = [0, 0, 3, 3, 3, 5, -1, 1, 0]
    want_k, want_v, whole = k.clone(), v.clone(), held.clone()
    got, got_lens, moves = paged.fork_pages(table, lens, numbers(parents), refs, k, v)
    want, want_lens, copies, lost = cache.fork(parents)
    assert not lost and got.tolist() == want and got_lens.tolist() == want_lens and refs.tolist() == cache.refs
    assert torch.equal(bits(k), bits(moved(want_k, copies))) and torch.equal(bits(v), bits(moved(want_v, copies)))
    # a cache in parts, by the moves
    parts = whole.clone()
    for layer in range(max(1, layers)):
        paged.copy_pages(*(t[layer] for t in paged.split_pages(parts, fmt)), moves[0], moves[1], moves[2])
    assert torch.equal(bits(parts), bits(held))
    paged.check_status()


def test_a_page_that_other_rows_hold_is_copied_for_every_writer():
    table, lens, refs = numbers([[3, 1]]), numbers([6]), numbers([0, 2, 0, 1, 0, 0])  # page 1 is also some other table's
    got, got_lens, moves = paged.fork_pages(table, lens, numbers([0, 0]), refs, page_size=4)
    assert got.tolist() == [[3, 0], [3, 2]] and moves.tolist() == [[1, 1], [0, 2], [2, 2]] and refs.tolist() == [1, 1, 1, 2, 0, 0]
    # a full last page is shared, whoever holds it
    refs = numbers([0, 2, 0, 1, 0, 0])
    got, _, moves = paged.fork_pages(table, numbers([8]), numbers([0, 0]), refs, page_size=4)
    assert got.tolist() == [[3, 1], [3, 1]] and moves.tolist() == [[-1, -1]] * 3 and refs.tolist() == [0, 3, 0, 2, 0, 0]


def test_without_a_free_page():
    paged.check_status()
    table, lens, refs = numbers([[0, 1]]), numbers([3]), numbers([1, 1, 0])
    got, got_lens, moves = paged.fork_pages(table, lens, numbers([0, 0, 0]), refs, page_size=2)
    assert got.tolist() == [[0, 1], [0, 2], [0, -1]] and got_lens.tolist() == [3, 3, 2] and refs.tolist() == [3, 1, 1]
    assert moves.tolist() == [[1, -1, -1], [2, -1, -1], [1, -1, -1]]
    with pytest.raises(RuntimeError, match="no free page"):
        paged.check_status()
    # the second row's pages are not there, the third needs none
    table, lens, refs = numbers([[0, -1, -1], [1, -1, -1], [2, -1, -1]]), numbers([2, 2, 1]), numbers([1, 1, 1, 0, 0])
    slots = paged.extend_pages(table, lens, refs, 2, q_starts=numbers([0, 1, 5, 6]), tokens=6)
    assert slots.tolist() == [6, -1, -1, -1, -1, 5] and table.tolist() == [[0, 3, -1], [1, -1, -1], [2, -1, -1]]
    assert lens.tolist() == [3, 2, 2] and refs.tolist() == [1, 1, 1, 1, 0]
    with pytest.raises(RuntimeError, match="no free page"):
        paged.check_status()


@pytest.mark.parametrize("rows,pages,page,width", SHAPES)
@pytest.mark.parametrize("kind", ["one", "some", "many"])
def test_extend(rows, pages, page, width, kind):
    rng = random.Random(rows + pages + len(kind))
    paged.check_status()
    cache, table, lens, refs = layout(rng, rows, pages, page, width, share=0.0, longest=max(1, min(width * page, pages * page // (3 * rows))))
    counts = [1 if kind == "one" else rng.choice([0, 1, 2, rng.randint(0, 3 * page + (900 if kind == "many" else 0))]) for _ in range(rows)]
    lead, tail = (0, 0) if kind == "one" else (2, 3)  # rows of no request
    starts = [lead]
    for c in counts:
        starts.append(starts[-1] + c)
    tokens = starts[-1] + tail
    want, without = cache.extend(counts, starts, tokens)
    got = paged.extend_pages(table, lens, refs, page) if kind == "one" else paged.extend_pages(table, lens, refs, page, numbers(starts), tokens)
    assert got.tolist() == want and table.tolist() == cache.table and lens.tolist() == cache.lens and refs.tolist() == cache.refs
    if without:
        with pytest.raises(RuntimeError):
            paged.check_status()
    paged.check_status()


@pytest.mark.parametrize("rows,pages,page,width", SHAPES)
def test_give_back(rows, pages, page, width):
    rng = random.Random(rows + pages)
    paged.check_status()
    cache, table, lens, refs = layout(rng, rows, pages, page, width, longest=max(1, min(width * page, pages * page // (2 * rows))))
    for some in ([], [rng.randrange(rows)], [-1] + rng.sample(range(rows), rows // 2) * 2):  # rows named twice are given back once
        paged.free_pages(table, lens, refs, page, rows=numbers(some, rng.choice([torch.int32, torch.int64])))
        cache.give_back(some)
        assert table.tolist() == cache.table and lens.tolist() == cache.lens and refs.tolist() == cache.refs
    paged.free_pages(table, lens, refs, page)
    assert not refs.any() and not lens.any() and (table == -1).all()
    paged.check_status()


@pytest.mark.parametrize("rows,pages,page,width", SHAPES)
@pytest.mark.parametrize("place", ["anywhere", "front", "back"])
def test_compact(rows, pages, page, width, place):
    rng = random.Random(rows + pages)
    cache, table, lens, refs = layout(rng, rows, pages, page, width, longest=max(1, min(width * page, pages * page // (2 * rows))))
    if place != "anywhere":  # held pages already at the front, or all at the back
        held = sorted({p for row, n in zip(cache.table, cache.lens) for p in row[:need(n, page)]})
        to = {p: i if place == "front" else pages - len(held) + i for i, p in enumerate(held)}
        cache = Cache(pages, page, [[to.get(p, -1) for p in row] for row in cache.table], cache.lens)
        table, refs = numbers(cache.table).view(rows, width), numbers(cache.refs)
    held, (k, v) = pool(2, pages, page if pages < 1000 else 1, 1, 8)
    before = k.clone(), v.clone()
    if pages < 1000:
        places, moves = paged.compact_pages(table, lens, refs, k, v)
    else:
        places, moves = paged.compact_pages(table, lens, refs, page_size=page)
        paged.copy_pages(k, v, moves[0], moves[1])
    want, copies = cache.compact()
    assert places.tolist() == want and refs.tolist() == cache.refs and table.tolist() == cache.table
    assert moves.tolist() == [[c[i] for c in copies] + [-1] * (pages // 2 - len(copies)) for i in range(2)]
    for t, b in zip((k, v), before):
        index = torch.arange(pages)
        for a, to in copies:
            index[to] = a
        assert torch.equal(bits(t), bits(b)[:, index.cuda()])
    paged.check_status()


@pytest.mark.parametrize("rows", [0, 3, 400])
def test_compact_of_a_large_cache(rows):
    """Copies by more blocks than run at a time, of which many, some or nearly all find nothing to do."""
    rng = random.Random(rows)
    pages, page = 12000, 2
    cache, table, lens, refs = layout(rng, rows, pages, page, 20, share=0.0)
    _, (k, v) = pool(2, pages, page, 1, 8)
    before = k.clone(), v.clone()
    places, moves = paged.compact_pages(table, lens, refs, k, v)
    want, copies = cache.compact()
    assert places.tolist() == want and refs.tolist() == cache.refs and table.tolist() == cache.table
    assert moves[:, :len(copies)].tolist() == [[c[i] for c in copies] for i in range(2)] and (moves[:, len(copies):] == -1).all()
    for t, b in zip((k, v), before):
        assert torch.equal(bits(t), bits(moved(b, [(a, to, page) for a, to in copies])) if copies else bits(b))
    paged.check_status()


@pytest.mark.parametrize("heads,head,page", [(8, 128, 16), (1, 128, 16), (3, 40, 5), (2, 7, 3), (12, 96, 24), (32, 128, 128)])
@pytest.mark.parametrize("fmt", ["vllm", "huggingface"])
@pytest.mark.parametrize("part", [False, True])
def test_copy(heads, head, page, fmt, part):
    rng = random.Random(page)
    held, (k, v) = pool(3, 23, page, heads, head, torch.bfloat16, fmt)
    order = rng.sample(range(23), 20)
    src, dst = order[:10], order[10:]
    src[3], dst[5] = -1, -1
    n = [rng.randint(0, page) if part else page for _ in src]
    want = [moved(t, [(a, b, m) for a, b, m in zip(src, dst, n) if a >= 0 and b >= 0]) for t in (k, v)]
    paged.copy_pages(k, v, numbers(src), numbers(dst), tokens=numbers(n) if part else None)
    assert torch.equal(bits(k), bits(want[0])) and torch.equal(bits(v), bits(want[1]))
    paged.check_status()


def test_copy_in_views_of_a_larger_array():
    """Strides and addresses that 16-byte accesses cannot take, and pages whose heads are part of wider ones."""
    big = torch.randint(-2 ** 15, 2 ** 15, (2, 11, 6, 4, 90), device="cuda", dtype=torch.int16).view(torch.float16)
    for cut in (slice(1, 65), slice(8, 72), slice(0, 89)):
        for heads in (slice(0, 4), slice(1, 2)):
            array = big.clone()
            k, v = array[0, :, :, heads, cut], array[1, :, 1:5, heads, cut][:, :4]
            k = k[:, :4]
            want = array.clone()
            for a, b in ((0, 5), (10, 2)):
                bits(want[0, :, :, heads, cut])[b, :4] = bits(array[0, :, :, heads, cut])[a, :4]
                bits(want[1, :, 1:5, heads, cut])[b, :4] = bits(array[1, :, 1:5, heads, cut])[a, :4]
            paged.copy_pages(k, v, numbers([0, 10]), numbers([5, 2]))
            assert torch.equal(bits(array), bits(want))


def test_copy_behind_4_gib():
    pages, page, head = 70, 64 * 1024, 512  # 4.4 GiB
    k = torch.zeros((pages, page, 1, head), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    k[68] = 3.0
    k[68, -1, 0, -1] = 7.0
    paged.copy_pages(k[..., :1], v[..., :1], numbers([68]), numbers([1]))
    assert (k[1, :, :, 0] == 3.0).all() and not k[1, :, :, 1:].any()
    paged.copy_pages(k, v, numbers([68]), numbers([69]))
    assert torch.equal(k[69], k[68]) and not v.any()


def test_pages_and_lengths_that_do_not_fit():
    paged.check_status()

    def flagged(text="slot, page or length"):
        with pytest.raises(RuntimeError, match=text):
            paged.check_status()

    _, (k, v) = pool(1, 4, 2, 1, 8)
    before = bits(k).clone()
    for src, dst, n in ((4, 1, 2), (1, 4, 2), (-2, 1, 2), (0, 1, 3), (0, 1, -1)):
        paged.copy_pages(k, v, numbers([src]), numbers([dst]), tokens=numbers([n]))
        assert torch.equal(bits(k), before)
        flagged()
    # a page that the cache does not have, and a row that is too long for its table: left out
    refs = numbers([1, 1, 0, 0])
    got, lens, _ = paged.fork_pages(numbers([[0, 9], [1, -1]]), numbers([4, 7]), numbers([0, 1]), refs, page_size=2, release=False)
    assert got.tolist() == [[0, -1], [1, -1]] and lens.tolist() == [4, 4] and refs.tolist() == [2, 2, 0, 0]
    flagged()
    got, lens, _ = paged.fork_pages(numbers([[0, 1]]), numbers([-3]), numbers([0, 1, -7]), numbers([1, 1, 0, 0]), page_size=2)
    assert got.tolist() == [[-1, -1]] * 3 and lens.tolist() == [0, 0, 0]
    flagged()
    # a page that nobody holds is not given back twice
    refs = numbers([1, 0, 0, 0])
    paged.free_pages(numbers([[0, 1]]), numbers([4]), refs, 2)
    assert not refs.any()
    flagged()
    paged.free_pages(numbers([[0, 1]]), numbers([0]), refs, 2, rows=numbers([1]))
    flagged()
    # tokens that a row's table has no room for, and starts that fall or lie outside
    table, lens, refs = numbers([[0], [1]]), numbers([2, 1]), numbers([1, 1, 0, 0])
    assert paged.extend_pages(table, lens, refs, 2, numbers([0, 1, 2]), 2).tolist() == [-1, 3]
    assert table.tolist() == [[0], [1]] and lens.tolist() == [2, 2] and refs.tolist() == [1, 1, 0, 0]
    flagged()
    paged.extend_pages(table, lens, refs, 2, numbers([2, 0, 9]), 2)
    flagged()
    assert table.tolist() == [[0], [1]] and lens.tolist() == [2, 2]
    table, refs = numbers([[0, 3]]), numbers([1, 0, 0, 0])
    paged.compact_pages(table, numbers([4]), refs, page_size=2)
    assert table.tolist() == [[0, 3]] and refs.tolist() == [1, 0, 0, 0]
    flagged()


def test_as_many_rows_as_a_call_takes():
    rows, pages, page = 4096, 30000, 4
    rng = random.Random(7)
    cache, table, lens, refs = layout(rng, rows, pages, page, 6, longest=20)
    parents = [rng.randrange(rows) for _ in range(rows)]
    got, got_lens, _ = paged.fork_pages(table, lens, numbers(parents), refs, page_size=page)
    cache.table, cache.lens, _, lost = cache.fork(parents)
    assert not lost and got.tolist() == cache.table and got_lens.tolist() == cache.lens and refs.tolist() == cache.refs
    counts = [rng.choice([0, 1, 1, 2]) for _ in range(rows)]
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    slots = paged.extend_pages(got, got_lens, refs, page, numbers(starts), starts[-1])
    before = list(cache.lens)
    want, without = cache_extend(cache, counts, starts)
    assert slots.tolist() == want and got.tolist() == cache.table and got_lens.tolist() == cache.lens and refs.tolist() == cache.refs
    assert without == [r for r in range(rows) if cache.lens[r] != before[r] + counts[r]]
    if without:
        with pytest.raises(RuntimeError):
            paged.check_status()
    paged.free_pages(got, got_lens, refs, page)
    assert not refs.any()
    paged.check_status()


def cache_extend(cache, counts, starts):
    """Cache.extend for many rows, without its sums over the rows in front."""
    slots, without, free, rank = [-1] * starts[-1], [], cache.free(), 0
    for r, c in enumerate(counts):
        before, after = need(cache.lens[r], cache.page), need(cache.lens[r] + c, cache.page)
        if after > len(cache.table[r]):
            without.append(r)
            continue
        first, rank = rank, rank + after - before
        if after > before and rank > len(free):
            without.append(r)
            continue
        for j in range(before, after):
            cache.table[r][j] = free[first + j - before]
            cache.refs[cache.table[r][j]] = 1
        for i in range(c):
            place = cache.lens[r] + i
            slots[starts[r] + i] = cache.table[r][place // cache.page] * cache.page + place % cache.page
        cache.lens[r] += c
    return slots, without


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_views_of_larger_arrays(offset):
    """Tables that are columns of wider ones, counts and lengths that begin inside an array: what stands beside them stays."""
    rng = random.Random(offset)
    for pages in (300, 9001):
        cache, table, lens, refs = layout(rng, 12, pages, 8, 9, longest=60)
        wide, tight, counts = torch.full((12, 20), 777, dtype=torch.int32, device="cuda"), torch.full((30,), 777, dtype=torch.int32, device="cuda"), torch.full((pages + 9,), 777, dtype=torch.int32, device="cuda")
        wide[:, offset:offset + 9], tight[offset:offset + 12], counts[offset:offset + pages] = table, lens, refs
        table, lens, refs = wide[:, offset:offset + 9], tight[offset:offset + 12], counts[offset:offset + pages]
        parents = [rng.randrange(12) for _ in range(12)]
        out = torch.full((12, 17), 777, dtype=torch.int32, device="cuda"), torch.full((12,), 777, dtype=torch.int32, device="cuda")
        got, got_lens, _ = paged.fork_pages(table, lens, numbers(parents), refs, page_size=8, out=(out[0][:, offset:offset + 9], out[1]))
        cache.table, cache.lens, _, lost = cache.fork(parents)
        assert not lost and got.tolist() == cache.table and got_lens.tolist() == cache.lens and refs.tolist() == cache.refs
        assert (out[0][:, :offset] == 777).all() and (out[0][:, offset + 9:] == 777).all()
        slots = paged.extend_pages(got, got_lens, refs, 8)
        want, without = cache.extend([1] * 12, list(range(13)), 12)
        assert slots.tolist() == want and got.tolist() == cache.table and refs.tolist() == cache.refs
        places, _ = paged.compact_pages(got, got_lens, refs, page_size=8)
        assert places.tolist() == cache.compact()[0] and got.tolist() == cache.table and refs.tolist() == cache.refs
        paged.free_pages(got, got_lens, refs, 8, rows=numbers([2, 5]))
        cache.give_back([2, 5])
        assert refs.tolist() == cache.refs and got.tolist() == cache.table
        for array, width in ((counts, pages), (tight, 12)):
            assert (array[:offset] == 777).all() and (array[offset + width:] == 777).all()
        assert (wide[:, :offset] == 777).all() and (wide[:, offset + 9:] == 777).all() and (out[0][:, offset + 9:] == 777).all()
        if without:
            with pytest.raises(RuntimeError):
                paged.check_status()
    paged.check_status()


def test_layers_of_one_array():
    """Keys and values that alternate in one array, layers and pages in any order of axes."""
    rng = random.Random(2)
    for axes in ((0, 1, 2, 3, 4, 5), (1, 2, 0, 3, 4, 5), (2, 0, 1, 4, 3, 5), (3, 0, 2, 1, 4, 5)):
        sizes = (3, 2, 25, 6, 4, 16)  # layers, keys and values, pages, tokens, heads, values
        array = torch.randint(-2 ** 15, 2 ** 15, [sizes[i] for i in axes], device="cuda", dtype=torch.int16).view(torch.bfloat16)
        cache = array.permute([axes.index(i) for i in range(6)])
        k, v = cache[:, 0], cache[:, 1]
        order = rng.sample(range(25), 16)
        n = [rng.randint(0, 6) for _ in range(8)]
        moves = list(zip(order[:8], order[8:], n))
        want = [moved(t, moves) for t in (k, v)]
        paged.copy_pages(k, v, numbers(order[:8]), numbers(order[8:]), tokens=numbers(n))
        assert torch.equal(bits(k), bits(want[0])) and torch.equal(bits(v), bits(want[1]))


def test_without_the_host_module(monkeypatch):
    """Through the general path: the same results, and the same errors as ever."""
    from cachegen_b200 import _lib, _plain_calls
    results = []
    for plain in (False, True):
        if plain:
            monkeypatch.setattr(_lib, "_calls", _plain_calls)
        rng = random.Random(3)
        cache, table, lens, refs = layout(rng, 6, 90, 4, 9, longest=30)
        _, (k, v) = pool(2, 90, 4, 2, 16)
        got, got_lens, moves = paged.fork_pages(table, lens, numbers([0, 0, 1, 4, 4, 5]), refs, k, v)
        slots = paged.extend_pages(got, got_lens, refs, 4, numbers([0, 2, 2, 9, 9, 10, 11]), 12)
        single = paged.extend_pages(got, got_lens, refs, 4)
        paged.free_pages(got, got_lens, refs, 4, rows=numbers([1, -1], torch.int64))
        places, more = paged.compact_pages(got, got_lens, refs, k, v)
        paged.copy_pages(k, v, numbers([3]), numbers([89]))
        g = torch.Generator(device="cuda").manual_seed(1)
        best = paged.beam_select(torch.randn((6, 999), generator=g, device="cuda"), -torch.arange(6.0, device="cuda").view(2, 3))
        results.append([got, got_lens, moves, slots, single, places, more, refs, bits(k), bits(v), *best])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    paged.check_status()


def test_nothing_to_do():
    e, refs, table = numbers([]), numbers([0, 1, 0]), torch.empty((0, 4), dtype=torch.int32, device="cuda")
    got, lens, moves = paged.fork_pages(table, e, e, refs, page_size=4)
    assert got.shape == (0, 4) and moves.shape == (3, 0)
    got, lens, moves = paged.fork_pages(numbers([[1, -1]]), numbers([3]), e, refs, page_size=4)  # all are given up
    assert got.shape == (0, 2) and refs.tolist() == [0, 0, 0]
    assert paged.extend_pages(table, e, refs, 4).shape == (0,)
    paged.free_pages(table, e, refs, 4)
    places, moves = paged.compact_pages(table, e, numbers([]), page_size=4)
    assert places.shape == (0,) and moves.shape == (2, 0)
    places, _ = paged.compact_pages(table, e, numbers([0, 5, 0]), page_size=4)
    assert places.tolist() == [-1, 0, -1]
    got, lens, _ = paged.fork_pages(torch.empty((1, 0), dtype=torch.int32, device="cuda"), numbers([0]), numbers([0, 0]), refs, page_size=4)
    assert got.shape == (2, 0) and lens.tolist() == [0, 0]
    k = torch.zeros((3, 2, 1, 8), dtype=torch.float16, device="cuda")
    paged.copy_pages(k, k.clone(), e, e)
    paged.check_status()


@pytest.mark.parametrize("seed", range(3))
def test_steps_together_leave_counts_that_match_the_tables(seed):
    rng = random.Random(seed)
    paged.check_status()
    pages, page, width, rows = 700, 8, 24, 20
    cache, table, lens, refs = layout(rng, rows, pages, page, width, longest=90)
    held, (k, v) = pool(2, pages, page, 2, 16)

    def tokens_of(row):
        return [bits(k)[0, cache.table[row][i // page], i % page, 0, 0].item() for i in range(cache.lens[row])]

    for _ in range(12):
        what = rng.choice(["fork", "extend", "free", "compact"])
        before = [tokens_of(r) for r in range(rows)]
        if what == "fork":
            parents = [rng.randrange(rows) for _ in range(rows)]
            table, lens, _ = paged.fork_pages(table, lens, numbers(parents), refs, k, v)
            cache.table, cache.lens, _, lost = cache.fork(parents)
            assert not lost
            before = [before[p] for p in parents]
        elif what == "extend":
            counts = [rng.randint(0, 3) for _ in range(rows)]
            starts = [sum(counts[:r]) for r in range(rows + 1)]
            slots = paged.extend_pages(table, lens, refs, page, numbers(starts), starts[-1])
            _, without = cache.extend(counts, starts, starts[-1])
            assert not without
            new = torch.randint(0, 999, (2, starts[-1], 2, 16), device="cuda", dtype=torch.int16).view(torch.float16)
            paged.append_paged(new, new.clone(), k, v, slots)
            before = [b + bits(new)[0, starts[r]:starts[r + 1], 0, 0].tolist() for r, b in enumerate(before)]
        elif what == "free":
            gone = rng.sample(range(rows), 3)
            paged.free_pages(table, lens, refs, page, rows=numbers(gone))
            cache.give_back(gone)
            before = [[] if r in gone else b for r, b in enumerate(before)]
        else:
            paged.compact_pages(table, lens, refs, k, v)
            cache.compact()
        assert table.tolist() == cache.table and lens.tolist() == cache.lens and refs.tolist() == cache.refs
        assert refs.tolist() == Cache(pages, page, cache.table, cache.lens).refs  # counted again from the tables
        assert [tokens_of(r) for r in range(rows)] == before  # every row still reads what it wrote
    paged.check_status()


def test_on_another_stream_and_in_a_graph():
    cache, table, lens, refs = layout(random.Random(5), 6, 80, 4, 10, longest=20)
    _, (k, v) = pool(1, 80, 4, 2, 16)
    parents = numbers([1, 1, 0, 4, 4, 2])
    paged.fork_pages(table, lens, parents, refs.clone(), k.clone(), v.clone())  # the status word, outside of the capture
    kept = [t.clone() for t in (table, lens, refs, k, v)]
    gone = numbers([3, -1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got, got_lens, moves = paged.fork_pages(table, lens, parents, refs, k, v)
        slots = paged.extend_pages(got, got_lens, refs, 4)
        paged.free_pages(got, got_lens, refs, 4, rows=gone)
        places, _ = paged.compact_pages(got, got_lens, refs, k, v)
    for _ in range(3):
        for t, was in zip((table, lens, refs, k, v), kept):
            t.copy_(was)
        graph.replay()
        want = Cache(80, 4, kept[0].tolist(), kept[1].tolist())
        k_want = kept[3].clone()
        want.table, want.lens, copies, _ = want.fork(parents.tolist())
        k_want = moved(k_want, copies)
        want_slots, _ = want.extend([1] * 6, list(range(7)), 6)
        want.give_back(gone.tolist())
        want_places, moves_ = want.compact()
        k_want = moved(k_want, [(a, b, 4) for a, b in moves_])
        assert slots.tolist() == want_slots and places.tolist() == want_places
        assert got.tolist() == want.table and got_lens.tolist() == want.lens and refs.tolist() == want.refs
        assert torch.equal(bits(k), bits(k_want))
    paged.check_status()

