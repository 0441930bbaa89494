"""Beam search on a paged cache: contexts appended, forked into beams, attended, chosen from, forked again and extended, step after step, with nothing
but calls of cachegen_b200.paged in between.  Keys and values are a function of a token and its place, so that at every step the cache of
each beam can be compared, bit for bit, with what its tokens, followed back on the host, say should be there."""
import math

import numpy as np
import pytest
import torch

from cachegen_b200 import paged
from pages_ref import Cache, best, need

pytestmark = pytest.mark.gpu


class Model:
    """One layer that looks tokens up, attends and looks the result up: no more than is needed for logits that depend on the whole sequence."""

    def __init__(self, vocab, heads, q_heads, head, dtype, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        new = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dtype)  # noqa: E731
        self.k, self.v, self.q = new(vocab, heads, head), new(vocab, heads, head), new(vocab, q_heads, head)
        self.places, self.out = new(512, heads, head), (torch.randn((q_heads * head, vocab), generator=g, device="cuda") * 0.5).to(dtype)

    def keys(self, tokens, places):
        return self.k[tokens] + self.places[places]

    def logits(self, attended):
        return attended.flatten(1) @ self.out


def attended_by_hand(model, q, tokens):
    """Attention of the last token over the whole sequence in 64 bits."""
    t, p = torch.tensor(tokens, device="cuda"), torch.arange(len(tokens), device="cuda")
    group = q.shape[0] // model.k.shape[1]
    k, v = model.keys(t, p).double().repeat_interleave(group, 1), model.v[t].double().repeat_interleave(group, 1)
    weights = torch.softmax(torch.einsum("hd,khd->hk", q.double(), k) / math.sqrt(q.shape[1]), -1)
    return torch.einsum("hk,khd->hd", weights, v)


def search(model, contexts, beams, steps, page, pages, width, check=True):
    """-> the beams' tokens and scores after every step"""
    dtype, (heads, head) = model.k.dtype, model.k.shape[1:]
    B, K = len(contexts), beams
    k_pages, v_pages = (torch.zeros((pages, page, heads, head), dtype=dtype, device="cuda") for _ in range(2))
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    table, lens = torch.full((B, width), -1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    # the contexts, as a decoder or a prompt's forward pass would bring them
    starts = np.cumsum([0] + [len(c) for c in contexts])
    slots = paged.extend_pages(table, lens, refs, page, torch.tensor(starts, dtype=torch.int32, device="cuda"), int(starts[-1]))
    tokens = torch.tensor([t for c in contexts for t in c], device="cuda")
    places = torch.tensor([i for c in contexts for i in range(len(c))], device="cuda")
    paged.append_paged(model.keys(tokens, places), model.v[tokens], k_pages, v_pages, slots)
    # each goes on in K beams, of which the first alone has begun
    table, lens, _ = paged.fork_pages(table, lens, torch.arange(B, device="cuda").repeat_interleave(K), refs, k_pages, v_pages)
    scores = torch.full((B, K), -math.inf, device="cuda")
    scores[:, 0] = 0.0
    sequences, newest, found = [list(c) for c in contexts for _ in range(K)], torch.tensor([c[-1] for c in contexts for _ in range(K)], device="cuda"), []
    for _ in range(steps):
        q = model.q[newest.clamp(min=0)]
        attended = paged.paged_attention(q, k_pages, v_pages, table, lens)
        logits = model.logits(attended)
        if check:
            for row in range(0, B * K, 3):
                if sequences[row] is not None:
                    want = attended_by_hand(model, q[row], sequences[row])
                    assert ((attended[row].double() - want).abs() <= 2e-2 * want.abs().max()).all()  # (what attention is off is tested elsewhere)
            want_scores, want_tokens, want_parents = best(logits.float().cpu().numpy(), scores.cpu().numpy(), K)
        scores, chosen, table, lens, slots = paged.beam_step(logits, scores, table, lens, refs, k_pages, v_pages)
        if check:
            assert np.array_equal(chosen.cpu().numpy(), want_tokens)
            there = np.isfinite(want_scores)
            assert np.allclose(scores.cpu().numpy()[there], want_scores[there], rtol=1e-6, atol=1e-5)
            sequences = [None if t < 0 else sequences[p] + [t] for p, t in zip(want_parents.ravel().tolist(), want_tokens.ravel().tolist())]
        newest = chosen.view(-1).long()
        paged.append_paged(model.keys(newest.clamp(min=0), (lens - 1).long()), model.v[newest.clamp(min=0)], k_pages, v_pages, slots)
        if check:
            rows, lengths = table.tolist(), lens.tolist()
            for row, tokens in enumerate(sequences):
                if tokens is None:
                    continue
                assert lengths[row] == len(tokens)
                at = torch.tensor([rows[row][i // page] * page + i % page for i in range(len(tokens))], device="cuda")
                k, v = paged.gather_paged(k_pages, v_pages, at)
                t, p = torch.tensor(tokens, device="cuda"), torch.arange(len(tokens), device="cuda")
                assert torch.equal(k, model.keys(t, p)) and torch.equal(v, model.v[t])
            assert refs.tolist() == Cache(pages, page, rows, lengths).refs  # counted again from the tables
        found.append((scores.clone(), chosen.clone(), table.clone(), lens.clone()))
    paged.free_pages(table, lens, refs, page)
    assert not refs.any()
    paged.check_status()
    return found


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page,beams,contexts", [(4, 4, (1, 9, 16)), (16, 8, (40, 3)), (1, 3, (5,)), (5, 1, (7, 7)), (64, 5, (130, 64, 63))])
def test_search(dtype, page, beams, contexts):
    model = Model(97, 2, 4, 32, dtype)
    g = torch.Generator().manual_seed(page)
    texts = [torch.randint(0, 97, (n,), generator=g).tolist() for n in contexts]
    width = need(max(contexts) + 12, page)
    search(model, texts, beams, 12, page, len(texts) * beams * width + 40, width)


def test_more_beams_than_continuations():
    model = Model(3, 1, 1, 16, torch.float16)  # three tokens: nine beams are not all begun before the third step
    search(model, [[0, 1], [2]], 9, 5, 2, 200, 8)


def test_the_same_in_a_graph():
    """Two steps, there and back between two sets of tables, captured and replayed, against the same steps one by one."""
    model, B, K, page, pages, width = Model(61, 2, 2, 32, torch.bfloat16), 2, 4, 4, 300, 12

    def begin():
        g = torch.Generator(device="cuda").manual_seed(3)
        state = dict(k=torch.randn((pages, page, 2, 32), generator=g, device="cuda").to(torch.bfloat16), v=torch.randn((pages, page, 2, 32), generator=g, device="cuda").to(torch.bfloat16),
                     refs=torch.zeros(pages, dtype=torch.int32, device="cuda"), tables=[torch.full((B * K, width), -1, dtype=torch.int32, device="cuda") for _ in range(2)],
                     lens=[torch.zeros(B * K, dtype=torch.int32, device="cuda") for _ in range(2)], scores=torch.zeros((B, K), device="cuda"),
                     newest=torch.arange(B * K, device="cuda"))
        starts = torch.arange(B * K + 1, dtype=torch.int32, device="cuda") * 6
        paged.extend_pages(state["tables"][0], state["lens"][0], state["refs"], page, starts, 6 * B * K)
        return state

    def steps(s):
        for i in range(2):
            attended = paged.paged_attention(model.q[s["newest"].clamp(min=0)], s["k"], s["v"], s["tables"][i], s["lens"][i])
            scores, chosen, _, lens, slots = paged.beam_step(model.logits(attended), s["scores"], s["tables"][i], s["lens"][i], s["refs"], s["k"], s["v"],
                                                             out=(s["tables"][1 - i], s["lens"][1 - i]))
            s["scores"].copy_(scores)
            s["newest"].copy_(chosen.view(-1))
            t = s["newest"].clamp(min=0)
            paged.append_paged(model.keys(t, (lens - 1).long()), model.v[t], s["k"], s["v"], slots)

    eager, replayed = begin(), begin()
    with torch.no_grad():
        warm = begin()
        steps(warm)
    kept = [t.clone() for t in (replayed["k"], replayed["v"], replayed["refs"], *replayed["tables"], *replayed["lens"], replayed["scores"], replayed["newest"])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(replayed)
    for t, was in zip((replayed["k"], replayed["v"], replayed["refs"], *replayed["tables"], *replayed["lens"], replayed["scores"], replayed["newest"]), kept):
        t.copy_(was)
    for _ in range(4):
        graph.replay()
        steps(eager)
        for name in ("refs", "scores", "newest", "k", "v"):
            assert torch.equal(eager[name], replayed[name]), name
        assert torch.equal(eager["tables"][0], replayed["tables"][0]) and torch.equal(eager["lens"][0], replayed["lens"][0])
    paged.check_status()


def test_a_context_from_the_codec_goes_on_in_beams():
    """A decoded context's tokens find their pages through extend_pages, and its beams share them."""
    from cachegen_b200.config import LMCacheEngineConfig, LMCacheEngineMetadata
    from cachegen_b200.serde import CacheGenDeserializer, CacheGenSerializer
    from cachegen_b200.synth import generate_kv
    L, H, D, T, page, pages = 32, 2, 64, 90, 16, 40
    engine, meta = LMCacheEngineConfig.from_defaults(chunk_size=256), LMCacheEngineMetadata("lmsys/longchat-7b-16k", 1, 0, "vllm")
    ser, de = CacheGenSerializer(engine, meta), CacheGenDeserializer(engine, meta, out_dtype=torch.float16)
    chunk = ser.encode(generate_kv(L, H, D, T, seed=3, device="cuda", dtype=torch.float16))
    want = de.decode(chunk)
    cache = torch.zeros((L, 2, pages, page, H, D), dtype=torch.float16, device="cuda")
    k_pages, v_pages = paged.split_pages(cache, "vllm")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    table, lens = torch.full((1, 8), -1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = paged.extend_pages(table, lens, refs, page, torch.tensor([0, T], dtype=torch.int32, device="cuda"), T)
    de.decode_paged([chunk], cache, slots)
    table, lens, _ = paged.fork_pages(table, lens, torch.zeros(4, dtype=torch.int32, device="cuda"), refs, k_pages, v_pages)
    rows = table.tolist()
    assert len({r[T // page] for r in rows}) == 4 and all(r[:T // page] == rows[0][:T // page] for r in rows)
    assert sorted(refs.tolist(), reverse=True)[:10] == [4] * 5 + [1] * 4 + [0]
    for row in rows:
        at = torch.tensor([row[i // page] * page + i % page for i in range(T)], device="cuda")
        k, v = paged.gather_paged(k_pages, v_pages, at)
        assert torch.equal(k, want[:, 0]) and torch.equal(v, want[:, 1])
    paged.check_status()
