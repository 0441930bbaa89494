"""Chunks to and from a paged cache, and the calls on it one after the other, as a serving program makes them."""
import math

import pytest
import torch

from paged_ref import attention, turned, turned_tolerance

pytestmark = pytest.mark.gpu

L, H, D, Q, PAGE = 32, 2, 64, 4, 16


@pytest.fixture(params=["vllm", "huggingface"])
def codec(request):
    from cachegen_b200.config import LMCacheEngineConfig, LMCacheEngineMetadata
    from cachegen_b200.serde import CacheGenDeserializer, CacheGenSerializer
    config = LMCacheEngineConfig.from_defaults(chunk_size=256)
    meta = LMCacheEngineMetadata(model_name="lmsys/longchat-7b-16k", world_size=1, worker_id=0, fmt=request.param)
    return CacheGenSerializer(config, meta), CacheGenDeserializer(config, meta, out_dtype=torch.float16), request.param


def blob(tokens, seed, fmt):
    from cachegen_b200.synth import generate_kv
    kv = generate_kv(L, H, D, tokens, seed=seed, device="cpu", dtype=torch.float16).cuda()
    return kv.permute(0, 1, 3, 2, 4).contiguous() if fmt == "huggingface" else kv


def new_pages(fmt, pages, dtype=torch.float16):
    shape = (L, 2, pages, PAGE, H, D) if fmt == "vllm" else (L, 2, pages, H, PAGE, D)
    return torch.full(shape, math.nan, dtype=dtype, device="cuda")


def rows(pages, fmt, slots):
    """Keys and values [L, tokens, H, D] that the pages have in these slots."""
    from cachegen_b200 import paged
    return [t[:, slots // PAGE, slots % PAGE] for t in paged.split_pages(pages, fmt)]


def test_a_context_in_and_out_of_pages(codec):
    """Bytes of two chunks into pages, bit for bit what from_bytes_many gives; and a range out of them, bit for bit what the same rows
    encode to."""
    ser, de, fmt = codec
    chunks = [blob(n, s, fmt) for n, s in ((200, 1), (57, 2))]
    blobs = [ser.to_bytes(c) for c in chunks]
    want = de.from_bytes_many(blobs)
    pages = new_pages(fmt, 20)
    slots = torch.randperm(20 * PAGE, generator=torch.Generator().manual_seed(3))[:257].cuda()
    for load in (lambda: de.from_bytes_paged(blobs, pages, slots), lambda: de.decode_paged([ser.encode(c) for c in chunks], pages, slots.int())):
        pages.fill_(math.nan)
        load()
        de.check_status()
        from cachegen_b200 import paged
        paged.check_status()
        for got, w in zip(rows(pages, fmt, slots), paged.split_blob(want, fmt)):
            assert torch.equal(got.view(torch.int16), w.contiguous().view(torch.int16))
        assert int(pages.isnan().sum()) == 2 * L * (20 * PAGE - 257) * H * D  # all else is as it was
    part = slots[30:130]
    again = ser.encode_paged(pages, part)
    same = ser.encode(want[:, :, 30:130].contiguous() if fmt == "vllm" else want[:, :, :, 30:130].contiguous())
    assert torch.equal(again.cdf, same.cdf) and torch.equal(again.data_chunks[0].bytestream, same.data_chunks[0].bytestream)
    assert torch.equal(again.max_tensors_key, same.max_tensors_key) and (again.num_heads, again.head_size) == (H, D)
    back = de.from_bytes(ser.to_bytes_paged(pages, part))
    assert torch.equal(back, de.decode(same))


def test_from_bytes_to_an_answer(codec):
    """A stored context without positions is loaded behind 1,000 others, new tokens are appended and attend to it, a chunk and then
    single tokens; each layer against the formulas in 64 bits on what stands in the pages."""
    from cachegen_b200 import paged
    ser, de, fmt = codec
    context, far, chunk = 203, 1000, 21
    kv = blob(context, 5, fmt)
    stored = ser.to_bytes(kv)
    decoded = de.from_bytes(stored)
    rotary = paged.Rotary(D, scaling=("linear", 2.0))
    pages = new_pages(fmt, 18)
    order = torch.randperm(18, generator=torch.Generator().manual_seed(6)).to(torch.int32).cuda()
    table = order[None]
    at = torch.arange(18 * PAGE, device="cuda")
    slots = order.long()[at // PAGE] * PAGE + at % PAGE
    de.from_bytes_paged([stored], pages, slots[:context], rotary=rotary, positions=far + at[:context])
    k0, v0 = (t.contiguous() for t in paged.split_blob(decoded, fmt))
    k_now, v_now = rows(pages, fmt, slots[:context])
    want = turned(k0, far + at[:context], rotary.frequencies, D, False)
    assert bool(((k_now.double() - want).abs() <= turned_tolerance(k0, want, D, False, torch.float16)).all()) and torch.equal(v_now, v0)
    k_pages, v_pages = paged.split_pages(pages, fmt)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    length = context
    for n in (chunk, 1, 1):
        place = slots[length:length + n]
        kv_lens = torch.tensor([length + n], dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        for layer in (0, 17, L - 1):
            q, k, v = (torch.randn((n, h, D), generator=g, device="cuda").half() for h in (Q, H, H))
            q = paged.append_paged(k, v, k_pages[layer], v_pages[layer], place, rotary=rotary, positions=far + at[length:length + n], q=q)
            out = paged.paged_attention(q, k_pages[layer], v_pages[layer], table, kv_lens, starts, max_q=n)
            w, _, tol = attention(q, k_pages[layer], v_pages[layer], table, [(0, n, length + n)], 1.0 / math.sqrt(D))
            assert bool(((out.double() - w).abs() <= tol).all())
        length += n
    paged.check_status()
    # out again without the positions, and moved to others
    k_back, _ = paged.gather_paged(k_pages, v_pages, slots[:context], rotary=rotary, positions=far + at[:context])
    unturned = turned(k_now, far + at[:context], rotary.frequencies, D, False, inverse=True)
    assert bool(((k_back.double() - unturned).abs() <= turned_tolerance(k_now, unturned, D, False, torch.float16)).all())
    moved = paged.apply_rotary(k_now, torch.full((context,), -250, device="cuda"), rotary)
    want = turned(k_now, torch.full((context,), -250, device="cuda"), rotary.frequencies, D, False)
    assert bool(((moved.double() - want).abs() <= turned_tolerance(k_now, want, D, False, torch.float16)).all())


def test_what_does_not_go_together_is_refused(codec):
    ser, de, fmt = codec
    chunk = ser.encode(blob(40, 1, fmt))
    pages, slots = new_pages(fmt, 4), torch.arange(40, device="cuda")
    for call, error in ((lambda: de.decode_paged([], pages, slots), RuntimeError), (lambda: de.decode_paged([chunk], pages, slots[:39]), RuntimeError),
                        (lambda: de.decode_paged([chunk], pages[:31], slots), RuntimeError), (lambda: de.decode_paged([chunk], pages[..., :32], slots), RuntimeError),
                        (lambda: de.decode_paged([chunk], pages.cpu(), slots), RuntimeError), (lambda: de.decode_paged([chunk], pages.float(), slots), RuntimeError),
                        (lambda: de.decode_paged([chunk], pages[:, :1], slots), RuntimeError),
                        (lambda: de.from_bytes_paged([chunk.to_bytes()], pages.bfloat16(), slots), TypeError),
                        (lambda: de.from_bytes_paged([chunk.to_bytes()], pages, slots[:39]), RuntimeError),
                        (lambda: ser.encode_paged(pages, slots[:0]), RuntimeError), (lambda: ser.encode_paged(pages[0], slots), RuntimeError),
                        (lambda: ser.encode_paged(pages.cpu(), slots), RuntimeError), (lambda: ser.to_bytes_paged(pages, slots[None]), RuntimeError)):
        with pytest.raises(error):
            call()


def test_without_the_native_calls_everything_is_the_same(monkeypatch):
    """The Python path of each call gives what the native one does."""
    from cachegen_b200 import _lib, _plain_calls, paged
    g = torch.Generator(device="cuda")
    g.manual_seed(1)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").half()
    rotary = paged.Rotary(64, rotary_dims=32, interleaved=True)
    x, q, k, v = rand(3, 9, 2, 64), rand(9, 4, 64), rand(9, 2, 64), rand(9, 2, 64)
    pages = rand(3, 2, 4, 8, 2, 64)
    slots, positions = torch.randperm(32, generator=torch.Generator().manual_seed(2))[:9].cuda(), torch.arange(9, device="cuda")
    table, lens = torch.tensor([[0, 3], [1, 2]], dtype=torch.int32, device="cuda"), torch.tensor([16, 9], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda")

    def everything():
        p = pages.clone()
        out = [paged.apply_rotary(x, positions, rotary), paged.apply_rotary(x, positions.expand(3, 9).contiguous(), rotary, inverse=True)]
        out.append(paged.append_paged(k, v, p[1, 0], p[1, 1], slots, rotary=rotary, positions=positions, q=q))
        assert paged.append_paged(x, x.clone(), p[:, 0], p[:, 1], slots.int()) is None
        out += [p, *paged.gather_paged(p[:, 0], p[:, 1], slots, rotary=rotary, positions=positions), *paged.gather_paged(p[2, 0], p[2, 1], slots)]
        out += paged.paged_attention(q, p[0, 0], p[0, 1], table, lens, starts, return_lse=True, window=7)
        out.append(paged.paged_attention(q[:2], p[0, 0], p[0, 1], table, lens, scale=0.3, out=torch.zeros_like(q[:2])))
        paged.check_status()
        return out
    taken = []
    calls = _lib.native_calls()
    for name in ("rotary", "append", "gather", "attend"):
        monkeypatch.setattr(calls, name, (lambda entry: lambda *a: (taken.append(entry(*a)), taken[-1])[1])(getattr(calls, name)))
    native = everything()
    assert len(taken) == 8 and all(t is not None for t in taken)
    monkeypatch.setattr(_lib, "_calls", _plain_calls)
    for a, b in zip(native, everything()):
        assert torch.equal(a, b)
