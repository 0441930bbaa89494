"""Rotary positions, append and gather on a paged cache against their formulas in 64 bits."""
import pytest
import torch

from paged_ref import turned, turned_tolerance

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_bad_pages():
    from cachegen_b200 import paged
    yield
    paged.check_status()


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def near(got, x, want, rot, interleaved):
    return bool(((got.double() - want).abs() <= turned_tolerance(x, want, rot, interleaved, got.dtype)).all())


def same(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


SHAPES = [  # lead, tokens, heads, head, rotary dims
    ((), 1, 1, 128, 128), ((), 37, 8, 128, 128), ((), 5, 3, 64, 32), ((), 9, 2, 80, 80), ((), 4, 1, 96, 48), ((3,), 17, 4, 128, 64),
    ((), 3, 2, 2, 2), ((), 6, 5, 7, 4), ((2,), 3, 3, 72, 40), ((), 3000, 8, 128, 128), ((33,), 130, 8, 128, 128), ((), 2, 300, 16, 16),
    ((), 2, 1, 512, 512), ((70000,), 1, 1, 16, 16), ((), 5000, 1, 128, 64), ((2,), 77, 1, 16, 16), ((), 1000, 3, 256, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead,tokens,heads,head,rot", SHAPES)
def test_rotary(lead, tokens, heads, head, rot, interleaved, dtype):
    from cachegen_b200 import paged
    r = paged.Rotary(head, rotary_dims=rot, interleaved=interleaved)
    x = randn(lead + (tokens, heads, head), dtype, 1)
    positions = torch.arange(11, 11 + tokens, device="cuda")
    want = turned(x, positions, r.frequencies, rot, interleaved)
    got = paged.apply_rotary(x, positions, r)
    assert near(got, x, want, rot, interleaved)
    assert same(got[..., rot:], x[..., rot:])
    again = x.clone()
    assert paged.apply_rotary(again, positions.int(), r, out=again) is again and same(again, got)  # in place
    back = paged.apply_rotary(x, positions, r, inverse=True)
    assert same(back, paged.apply_rotary(x, positions, r, inverse=1))
    assert near(back, x, turned(x, positions, r.frequencies, rot, interleaved, inverse=True), rot, interleaved)


@pytest.mark.parametrize("position", [0, -1, -123456, 999_983, 2 ** 31 - 1, 2 ** 31 + 12345, 2 ** 40 + 7])
@pytest.mark.parametrize("scaling", [None, ("linear", 8.0), ("ntk", 4.0), ("bands", 8.0, 1.0, 4.0, 8192)])
def test_far_positions_and_scaled_frequencies(position, scaling):
    from fractions import Fraction
    from cachegen_b200 import paged
    r = paged.Rotary(64, base=500000.0, scaling=scaling)
    x = randn((1, 2, 64), torch.bfloat16, 2)
    # an angle of 2^40 radians has 13 bits behind its point in 64: whole turns are taken off in exact arithmetic
    turn = paged._TWO_PI
    reduced = [float(Fraction(f) * position - int(Fraction(f) * position / turn) * turn) for f in r.frequencies]
    want = turned(x, torch.ones(1, device="cuda"), reduced, 64, False)
    got = paged.apply_rotary(x, torch.tensor([position], device="cuda"), r)
    assert near(got, x, want, 64, False)


def test_given_frequencies_and_positions_a_layer():
    from cachegen_b200 import paged
    w = [1.5, 7.0, -0.25, 0.0]
    r = paged.Rotary(16, rotary_dims=8, frequencies=w)
    x = randn((4, 6, 3, 16), torch.float16, 3)
    positions = torch.arange(24, device="cuda").view(4, 6)
    assert near(paged.apply_rotary(x, positions, r), x, turned(x, positions, w, 8, False), 8, False)


def test_strided_rows_and_odd_addresses():
    from cachegen_b200 import paged
    r = paged.Rotary(64)
    base = randn((9, 5, 3 * 64 + 2), torch.float16, 4)
    positions = torch.arange(9, device="cuda")
    for x in (base[:, ::2, 64:128], base[:, :, 1:65], base.transpose(0, 1)[:4, :, :64].transpose(0, 1)):
        out = torch.zeros((9, x.shape[1], 70), dtype=torch.float16, device="cuda")
        got = paged.apply_rotary(x, positions, r, out=out[:, :, 3:67])
        assert near(got, x, turned(x, positions, r.frequencies, 64, False), 64, False)
        assert not out[:, :, :3].any() and not out[:, :, 67:].any()


CACHES = [  # layers (0: no axis), tokens, q heads, heads, head, rot, page, heads before tokens
    (0, 1, 4, 1, 128, 128, 16, False), (0, 64, 32, 8, 128, 128, 16, False), (0, 33, 4, 4, 80, 80, 24, True), (0, 19, 0, 3, 64, 0, 1, False),
    (3, 50, 0, 8, 128, 128, 16, True), (32, 131, 0, 4, 128, 64, 64, False), (0, 7, 6, 2, 40, 20, 5, False), (2, 700, 0, 8, 128, 128, 8, False),
    (0, 2048, 32, 32, 64, 64, 128, True)]


def cache(layers, pages, page, heads, head, dtype, transposed, seed):
    lead = (layers,) if layers else ()
    t = randn(lead + (2, pages) + ((heads, page) if transposed else (page, heads)) + (head,), dtype, seed)
    t = t.transpose(-2, -3) if transposed else t
    return t.unbind(-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layers,tokens,q_heads,heads,head,rot,page,transposed", CACHES)
def test_append_and_gather(layers, tokens, q_heads, heads, head, rot, page, transposed, interleaved, dtype):
    from cachegen_b200 import paged
    r = paged.Rotary(head, rotary_dims=rot, interleaved=interleaved) if rot else None
    lead = (layers,) if layers else ()
    pages = (tokens + page - 1) // page + 2
    kp, vp = cache(layers, pages, page, heads, head, dtype, transposed, 5)
    kp0, vp0 = kp.clone(), vp.clone()
    k, v = (randn(lead + (tokens, heads, head), dtype, s) for s in (6, 7))
    q = randn((tokens, q_heads, head), dtype, 8) if q_heads else None
    g = torch.Generator()
    g.manual_seed(9)
    slots = torch.randperm(pages * page, generator=g)[:tokens].cuda()
    padding = torch.arange(tokens, device="cuda") % 7 == 3
    slots[padding] = -1
    positions = torch.arange(1000, 1000 + tokens, device="cuda")
    out = torch.full_like(q, 5.0) if q_heads else None
    got = paged.append_paged(k, v, kp, vp, slots, rotary=r, positions=positions if r else None, q=q, q_out=out)
    assert got is out
    w = r.frequencies if r else []
    page_of, in_page = slots[~padding] // page, slots[~padding] % page
    k_want = turned(k, positions, w, rot, interleaved)[..., ~padding, :, :]
    assert near(kp[..., page_of, in_page, :, :], k[..., ~padding, :, :], k_want, rot, interleaved)
    assert same(vp[..., page_of, in_page, :, :], v[..., ~padding, :, :])
    if q_heads:
        q_want = turned(q, positions, w, rot, interleaved)
        assert near(out[~padding], q[~padding], q_want[~padding], rot, interleaved) and bool((out[padding] == 5.0).all())
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots[~padding]] = False
    rest = rest.nonzero()[:, 0]
    for now, was in ((kp, kp0), (vp, vp0)):  # all other slots are as they were
        assert same(now[..., rest // page, rest % page, :, :], was[..., rest // page, rest % page, :, :])
    stored = kp.clone()
    k_back, v_back = (torch.full_like(t, 3.0) for t in (k, v))
    paged.gather_paged(kp, vp, slots.int(), k=k_back, v=v_back, rotary=r, positions=positions if r else None)
    seen = stored[..., page_of, in_page, :, :]
    want = turned(seen, positions[~padding], w, rot, interleaved, inverse=True)
    assert near(k_back[..., ~padding, :, :], seen, want, rot, interleaved) and same(v_back[..., ~padding, :, :], v[..., ~padding, :, :])
    assert bool((k_back[..., padding, :, :] == 3.0).all()) and bool((v_back[..., padding, :, :] == 3.0).all())
    assert same(kp, stored)
    k_new, v_new = paged.gather_paged(kp, vp, slots[~padding])
    assert same(k_new, seen) and same(v_new, v_back[..., ~padding, :, :])


def test_copies_keep_every_bit():
    """NaN payloads, infinities, negative zero: what is not rotated is not computed with."""
    from cachegen_b200 import paged
    bits = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16)
    for dtype in TYPES:
        v = bits.view(dtype).view(64, 8, 128)
        k_pages, v_pages = (torch.zeros((16, 4, 8, 128), dtype=dtype, device="cuda") for _ in range(2))
        slots = torch.arange(64, device="cuda").flip(0)
        paged.append_paged(v, v, k_pages, v_pages, slots)
        assert same(v_pages.view(64, 8, 128).flip(0), v) and same(k_pages.view(64, 8, 128).flip(0), v)


def test_slots_outside_the_cache_are_left_out_and_reported():
    from cachegen_b200 import paged
    k, v = (randn((6, 2, 64), torch.float16, s) for s in (1, 2))
    kp, vp = (torch.zeros((3, 4, 2, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    slots = torch.tensor([0, 12, -2, 2 ** 40, 11, -1], device="cuda")
    paged.append_paged(k, v, kp, vp, slots)
    with pytest.raises(RuntimeError, match="paged cache"):
        paged.check_status()
    paged.check_status()
    assert same(kp[0, 0], k[0]) and same(vp[2, 3], v[4]) and int(kp.ne(0).any(-1).any(-1).sum()) == 2
    out = torch.full((6, 2, 64), 2.0, dtype=torch.float16, device="cuda")
    paged.gather_paged(kp, vp, slots, k=out, v=out.clone())
    with pytest.raises(RuntimeError, match="paged cache"):
        paged.check_status()
    assert same(out[0], k[0]) and same(out[4], k[4]) and bool((out[[1, 2, 3, 5]] == 2.0).all())


def test_offsets_beyond_32_bits():
    """Pages of one array that lie more than 2^31 values apart."""
    from cachegen_b200 import paged
    store = torch.zeros(2 ** 31 + 2 ** 21, dtype=torch.float16, device="cuda")
    kp = store.as_strided((3, 4, 2, 64), (2 ** 30, 128, 64, 1))
    vp = store.as_strided((3, 4, 2, 64), (2 ** 30, 128, 64, 1), 2 ** 20)
    k, v = (randn((12, 2, 64), torch.float16, s) for s in (1, 2))
    slots = torch.arange(12, device="cuda").flip(0)
    paged.append_paged(k, v, kp, vp, slots)
    assert same(kp.reshape(12, 2, 64).flip(0), k) and same(vp.reshape(12, 2, 64).flip(0), v)
    k2, v2 = paged.gather_paged(kp, vp, slots)
    assert same(k2, k) and same(v2, v)


def test_nothing_to_do():
    from cachegen_b200 import paged
    r = paged.Rotary(64)
    none = torch.empty((0, 2, 64), dtype=torch.float16, device="cuda")
    at = torch.empty(0, dtype=torch.int64, device="cuda")
    assert paged.apply_rotary(none, at, r).shape == (0, 2, 64)
    kp = torch.ones((3, 4, 2, 64), dtype=torch.float16, device="cuda")
    paged.append_paged(none, none, kp, kp.clone(), at, rotary=r, positions=at)
    assert bool((kp == 1).all())
    assert paged.gather_paged(kp, kp, at)[0].shape == (0, 2, 64)


def test_another_stream_and_a_graph():
    from cachegen_b200 import paged
    r = paged.Rotary(128)
    k, v, q = (randn((16, h, 128), torch.bfloat16, h) for h in (2, 3, 8))
    v = v[:, :2].contiguous()
    kp, vp = (torch.zeros((4, 16, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots, positions = torch.arange(16, device="cuda"), torch.arange(50, 66, device="cuda")
    want_q = paged.append_paged(k, v, kp, vp, slots, rotary=r, positions=positions, q=q)
    want_k, want_v = kp[0].clone(), vp[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kp.zero_()
        out = paged.append_paged(k, v, kp, vp, slots + 16, rotary=r, positions=positions, q=q)
    side.synchronize()
    assert same(kp[1], want_k) and same(vp[1], want_v) and same(out, want_q) and not kp[0].any()
    graph = torch.cuda.CUDAGraph()
    moved, place = slots.clone(), positions.clone()
    with torch.cuda.graph(graph):
        out = paged.append_paged(k, v, kp, vp, moved, rotary=r, positions=place, q=q)
        back = paged.gather_paged(kp, vp, moved, rotary=r, positions=place)
    for shift in (32, 48):
        moved.copy_(slots + shift)
        graph.replay()
        assert same(kp[shift // 16], want_k) and same(out, want_q) and same(back[1], want_v)
    place.copy_(positions + 5)
    graph.replay()
    assert near(kp[3], k, turned(k, positions + 5, r.frequencies, 128, False), 128, False)
