"""Beam search on a paged KV cache, and the pages that requests share, as measurable cases.

A case is one call of a public entry point of cachegen_b200.paged:

    select    beam_select                   the best continuations of every request's beams over the whole vocabulary
    fork      fork_pages                    tables of new rows that go on from given ones: pages shared, last ones copied
    copy      copy_pages                    pages (or the first tokens of them) copied to other places of the cache
    compact   compact_pages                 held pages moved to the front of the cache, tables after them
    turnover  free_pages and extend_pages   requests that have ended leave, others come in their places, all get room for their next tokens

    dtype            float16, bfloat16, or (logits) float32
    batch, beams     requests, and beams of each (select, fork); batch alone: rows of the table (compact, turnover)
    vocab, k         tokens of the vocabulary, continuations chosen for a request; pad: values between two rows of logits
    banned           share of the tokens whose logits are -infinity; first: only the first beam of a request has begun
    layers, heads, head, page    the cache: layers (0: one layer's tensors without an axis for it), heads, values of a head, tokens of a page
    context, ragged  tokens of the longest row, and how far the others may fall short of it (a share)
    release          the new rows take the old ones' place (a step of beam search); else the old ones stay (continuations of a context)
    pages, part      pages to copy; whether only their first tokens are
    spread           share of the cache's pages that are held
    ended, prompt    share of the rows that end, tokens of the longest that comes

The plain forms here are elementary torch operations.  Scores are worked out in 64 bits, since continuations that lie close together
in them would change places in 32, and rounded once; everything else is whole numbers and copies.
"""
import json
import math
import random

import numpy as np
import torch

own = False  # False: the plain forms; True: the calls of cachegen_b200.paged

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def _case(name, op, **given):
    case = {"op": op, "dtype": "bfloat16", "batch": 1, "beams": 1, "vocab": 32000, "k": 1, "pad": 0, "banned": 0.0, "first": False,
            "layers": 32, "heads": 8, "head": 128, "page": 16, "context": 1, "ragged": 0.0, "release": True, "pages": 1, "part": False,
            "spread": 0.5, "ended": 0.0, "prompt": 1}
    case.update(given)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # a step of one request with four beams: a call whose time is its launches
        _case("select_1x4", "select", beams=4, k=8, dtype="float16"),
        # the first step of a few requests with a vocabulary of odd size: all beams but the first are still empty
        _case("select_8x5_first", "select", batch=8, beams=5, vocab=50257, k=10, first=True),
        # answers held to a grammar, logits in 32 bits, as a head that keeps its sums gives them
        _case("select_16x16_banned", "select", batch=16, beams=16, vocab=65537, k=32, banned=0.9, dtype="float32", pad=7),
        # a step of a full batch with a large vocabulary
        _case("select_64x8", "select", batch=64, beams=8, vocab=128000, k=16),
        # one request's context, just loaded, goes on in four ways: latency
        _case("fork_context_61", "fork", beams=4, context=61, layers=10, release=False),
        # a step of a full batch of beams over the cache of one shard's layers
        _case("fork_beams_64x8", "fork", batch=64, beams=8, context=2048, ragged=0.7, layers=10),
        # a few pages of one layer
        _case("copy_5", "copy", pages=5, layers=0),
        # the last pages of many contexts to pages of their own, heads' tokens side by side, odd head size
        _case("copy_parts_700", "copy", pages=700, layers=10, heads=8, head=80, page=64, part=True, dtype="float16"),
        # a small cache of one shard's layers, nearly full
        _case("compact_300", "compact", batch=12, context=400, ragged=0.5, layers=10, heads=1, spread=0.9),
        # a larger one from which half of the requests have gone
        _case("compact_4096", "compact", batch=64, context=600, ragged=0.5, layers=10, spread=0.5),
        # the end of a step of eight requests: one leaves, another comes
        _case("turnover_8", "turnover", batch=8, context=3000, ragged=0.8, ended=0.12, prompt=500),
        # the same of a full cache of small pages
        _case("turnover_512", "turnover", batch=512, context=4096, ragged=0.9, ended=0.1, prompt=2000, page=8, spread=0.8),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


_MOST_LOGITS, _MOST_CACHE, _MOST_MOVED = 131_000_000, 4 << 30, 1_180_000_000  # bytes of a drawn case


def draw(rng):
    op = rng.choice(["select", "select", "select", "fork", "fork", "copy", "compact", "turnover"])
    if op == "select":
        case = _case(None, op, dtype=rng.choice(sorted(_DTYPES)), batch=_log(rng, 1, 64), beams=_log(rng, 1, 32),
                     vocab=_log(rng, 1000, 260000), pad=rng.choice([0, 0, 1, 8]), banned=rng.choice([0.0, 0.0, 0.3, 0.99]),
                     first=rng.random() < 0.2)
        case["k"] = rng.choice([case["beams"], 2 * case["beams"], _log(rng, 1, 64)])
        while work(case)["bytes"] > _MOST_LOGITS:
            case["batch" if case["batch"] > 1 else "vocab"] //= 2
        return case
    heads, head = rng.choice([(8, 128), (8, 128), (32, 128), (4, 128), (1, 128), (8, 64), (8, 80), (12, 96)])
    case = _case(None, op, dtype=rng.choice(["float16", "bfloat16"]), heads=heads, head=head, page=rng.choice([16, 16, 64, 32, 128, 8, 24]),
                 layers=rng.choice([0, 1, 10, 32, 80]), context=_log(rng, 1, 8192), ragged=rng.choice([0.0, 0.3, 0.9]))
    if op == "fork":
        case.update(batch=_log(rng, 1, 64), beams=_log(rng, 1, 8), release=rng.random() < 0.7)
    elif op == "copy":
        case.update(pages=_log(rng, 1, 2000), part=rng.random() < 0.5)
    else:
        case.update(batch=_log(rng, 1, 64 if op == "compact" else 512), spread=rng.choice([0.3, 0.6, 0.9]))
    if op == "turnover":
        case.update(ended=rng.choice([0.0, 0.1, 0.5, 1.0]), prompt=_log(rng, 1, 8192))
        return case
    while _pool(case) * _page_bytes(case) > _MOST_CACHE or work(case)["bytes"] > _MOST_MOVED:
        at = "pages" if op == "copy" else "batch" if case["batch"] > 1 else "context"
        if case[at] > 1:
            case[at] = (case[at] + 1) // 2
        else:
            case["layers"] = case["layers"] // 2 or 1
            case["page"] = min(case["page"], 16)
    return case


def _page_bytes(case):
    """Of keys and values of every layer."""
    return 2 * 2 * max(1, case["layers"]) * case["page"] * case["heads"] * case["head"]


def _shape_of(case):
    """What does not depend on a seed, the same for the same case."""
    return random.Random(json.dumps({n: v for n, v in sorted(case.items()) if n != "name"}))


def _lengths(case, rng):
    """Lengths of rows: the first is the longest, the others fall short by up to `ragged`."""
    return [max(1, int(case["context"] * (1.0 - rng.random() * case["ragged"] * (i > 0)))) for i in range(case["batch"])]


def _need(n, page):
    return (n + page - 1) // page


def _layout(case):
    """Rows as (length, [places in the cache's order of use]), places in use, places in all, and what else a case has."""
    rng, page = _shape_of(case), case["page"]
    lens = _lengths(case, rng)
    rows, used, more = [], 0, {}
    beams = case["beams"] if case["op"] == "fork" and case["release"] else 1
    for n in lens:
        pages = _need(n, page)
        common = rng.randrange(max(0, pages - 6), pages) if beams > 1 else 0  # beams share a context's pages up to where they part
        for b in range(beams):
            mine = list(range(used, used + (pages if b == 0 else pages - common)))
            rows.append((n, mine if b == 0 else rows[-b][1][:common] + mine))
            used += len(mine)
    if case["op"] == "fork":
        many = case["beams"]
        if case["release"]:  # a step's parents: the better beams go on more often
            more["parents"] = [i * many + min(int(many * rng.random() ** 1.5), many - 1) for i in range(case["batch"]) for _ in range(many)]
        else:
            more["parents"] = [i for i in range(case["batch"]) for _ in range(many)]
        total = used + len(more["parents"]) + used // 8 + 3
    elif case["op"] == "turnover":
        more["ended"] = [i for i in range(len(rows)) if rng.random() < case["ended"]]
        more["new"] = [1] * len(rows)
        for i in more["ended"]:
            more["new"][i] = max(1, int(case["prompt"] * rng.random()))
        comes = sum(_need(n, page) + 1 for n in more["new"])
        total = max(int(used / case["spread"]), used + comes) + 1
    else:
        total = int(used / case["spread"]) + 1
    return rows, used, total, more


def _pool(case):
    return 2 * case["pages"] + 3 if case["op"] == "copy" else _layout(case)[2]


def _parts(case):
    """Tokens copied of each page."""
    rng = _shape_of(case)
    return [rng.randint(1, case["page"]) if case["part"] else case["page"] for _ in range(case["pages"])]


def _copies(case, rows, parents):
    """Of a fork: (new row, tokens) of the last pages that have to be copied."""
    seen, out = set(), []
    for i, p in enumerate(parents):
        tokens = rows[p][0] % case["page"]
        if tokens and (p in seen or not case["release"]):
            out.append((i, tokens))
        seen.add(p)
    return out


def work(case):
    if case["op"] == "select":
        size = 4 if case["dtype"] == "float32" else 2
        rows = case["batch"] * (1 if case["first"] else case["beams"])
        return {"bytes": rows * case["vocab"] * size + 4 * case["batch"] * (case["beams"] + 3 * case["k"]), "flops": 3 * rows * case["vocab"]}
    token = _page_bytes(case) // case["page"]
    if case["op"] == "copy":
        return {"bytes": 2 * token * sum(_parts(case)) + 3 * 8 * case["pages"], "flops": case["pages"]}
    rows, used, total, more = _layout(case)
    entries = sum(len(p) for _, p in rows)
    if case["op"] == "fork":
        moved = sum(n for _, n in _copies(case, rows, more["parents"]))
        new = sum(len(rows[p][1]) for p in more["parents"])
        return {"bytes": 2 * token * moved + 4 * (entries + new + 2 * total), "flops": entries + new}
    if case["op"] == "compact":
        moved = used * (total - used) // total  # about: of pages in any order, those behind the `used`-th
        return {"bytes": 2 * token * case["page"] * moved + 4 * (2 * entries + 3 * total), "flops": entries + total}
    gone = sum(len(rows[i][1]) for i in more["ended"])
    return {"bytes": 4 * (2 * gone + 2 * total + 4 * len(rows)) + 8 * sum(more["new"]), "flops": gone + total}


def _normal(g, shape, dtype):
    """Values as a model's projections give them: channels of unlike scale."""
    scale = torch.exp(0.4 * torch.randn(shape[-2:], generator=g, device="cuda"))
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1, *shape[-2:])
    step = max(1, (1 << 26) // max(1, flat[0].numel()))
    for at in range(0, flat.shape[0], step):
        part = flat[at:at + step]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * scale)
    return out


def _cache(case, g, pool):
    lead = (case["layers"],) if case["layers"] else ()
    return [_normal(g, lead + (pool, case["page"], case["heads"], case["head"]), _DTYPES[case["dtype"]]) for _ in range(2)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = {"case": case}
    if case["op"] == "select":
        B, K, V = case["batch"], case["beams"], case["vocab"]
        # logits as a head gives them: a broad bulk, and a few tokens of each row that stand out
        logits = 2.2 * torch.randn((B * K, V), generator=g, device="cuda")
        tops = torch.randint(0, V, (B * K, 24), generator=g, device="cuda")
        logits.scatter_add_(1, tops, 4.0 + 3.0 * torch.rand(tops.shape, generator=g, device="cuda"))
        if case["banned"]:
            logits.masked_fill_(torch.rand((B * K, V), generator=g, device="cuda") < case["banned"], -math.inf)
        held = torch.zeros((B * K, V + case["pad"]), dtype=_DTYPES[case["dtype"]], device="cuda")
        held[:, :V] = logits
        state["logits"] = held[:, :V]
        scores = -20.0 * torch.rand((B, K), generator=g, device="cuda")
        if case["first"]:
            scores[:, 1:] = -math.inf
            scores[:, 0] = 0.0
        state["scores"] = scores
        return state
    draw_from = np.random.RandomState(seed % (1 << 32))
    if case["op"] == "copy":
        order = draw_from.permutation(_pool(case))
        n = case["pages"]
        state["src"], state["dst"] = (torch.from_numpy(order[k * n:k * n + n].astype(np.int64)).cuda() for k in range(2))
        state["tokens"] = torch.tensor(_parts(case), dtype=torch.int32, device="cuda") if case["part"] else None
        state["pages"] = _cache(case, g, _pool(case))
        return state
    rows, used, total, more = _layout(case)
    order = draw_from.permutation(total).astype(np.int32)
    longest = max(len(p) for _, p in rows)
    if case["op"] == "turnover":
        longest = max([longest + 1] + [_need(n, case["page"]) for n in more["new"]])
    table = np.full((len(rows), longest), -1, dtype=np.int32)
    for i, (_, pages) in enumerate(rows):
        table[i, :len(pages)] = order[pages]
    counts = np.bincount(table[table >= 0], minlength=total).astype(np.int32)
    lens = np.array([n for n, _ in rows], dtype=np.int32)
    # what the calls change in place is parts of one array, put back in front of every pass
    state["as_it_was"] = torch.from_numpy(np.concatenate([counts, lens, table.ravel()])).cuda()
    live = state["as_it_was"].clone()
    state["live"] = live
    state["refs"], state["lens"] = live[:total], live[total:total + len(rows)]
    state["table"] = live[total + len(rows):].view(len(rows), longest)
    if case["op"] == "fork":
        state["parents"] = torch.tensor(more["parents"], dtype=torch.int32, device="cuda")
        state["pages"] = _cache(case, g, total)
    elif case["op"] == "compact":
        state["pages"] = _cache(case, g, total)
    else:
        starts = np.concatenate([[0], np.cumsum(more["new"])]).astype(np.int32)
        state["ended"] = torch.tensor(more["ended"], dtype=torch.int64, device="cuda")
        state["starts"], state["tokens"] = torch.from_numpy(starts).cuda(), int(starts[-1])
    return state


def _pages_held(table, lens, page):
    """Which entries of a table stand for pages that its rows hold."""
    return torch.arange(table.shape[1], device=table.device) < ((lens + (page - 1)) // page)[:, None]


def _how_often(entries, total):
    return torch.zeros(total, dtype=torch.int32, device=entries.device).scatter_add_(
        0, entries.long(), torch.ones_like(entries, dtype=torch.int32))


def _free_ones(refs):
    """Numbers of the pages, free ones in front, lowest first."""
    return torch.sort((refs != 0).to(torch.int32), stable=True).indices


def _plain_copy(pages, src, dst, tokens, page):
    for t in pages:
        lead = t.dim() - 4
        at = (slice(None),) * lead
        if tokens is None:
            t[at + (dst,)] = t[at + (src,)]
        else:
            i, j = torch.nonzero(torch.arange(page, device=t.device) < tokens[:, None], as_tuple=True)
            t[at + (dst[i], j)] = t[at + (src[i], j)]


def _plain_select(s):
    case, logits, scores = s["case"], s["logits"], s["scores"]
    B, K, V, k = case["batch"], case["beams"], case["vocab"], case["k"]
    flat = torch.empty((B, K * V), dtype=torch.float64, device=logits.device)
    for b in range(B):
        x = logits[b * K:(b + 1) * K].double()
        top = x.amax(-1, keepdim=True)
        flat[b] = (scores[b].double()[:, None] + (x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True)))).view(-1)
    least = torch.topk(flat, min(k, K * V), dim=-1).values[:, -1:]
    b, i = torch.nonzero((flat >= least) & (flat > -math.inf), as_tuple=True)  # of equal ones more than k may be left
    value = flat[b, i]
    order = torch.sort(value, descending=True, stable=True).indices  # by request, then by score, then by index
    order = order[torch.sort(b[order], stable=True).indices]
    b, i, value = b[order], i[order], value[order]
    place = torch.arange(b.numel(), device=b.device) - torch.searchsorted(b, torch.arange(B, device=b.device))[b]
    b, i, value, place = (t[place < k] for t in (b, i, value, place))
    got = torch.full((B, k), -math.inf, dtype=torch.float32, device=b.device)
    tokens, parents = (torch.full((B, k), -1, dtype=torch.int32, device=b.device) for _ in range(2))
    got[b, place] = value.float()
    tokens[b, place], parents[b, place] = (i % V).to(torch.int32), (b * K + i // V).to(torch.int32)
    return [got, tokens, parents]


def _plain_fork(s):
    case, refs, table, lens, parents, page = s["case"], s["refs"], s["table"], s["lens"], s["parents"].long(), s["case"]["page"]
    P, N = refs.shape[0], parents.shape[0]
    new_lens = lens[parents]
    held = _pages_held(table, lens, page)
    new_held = held[parents]
    new = torch.where(new_held, table[parents], -1)
    refs += _how_often(new[new_held], P)
    if case["release"]:
        refs -= _how_often(table[held], P)
    part, last = new_lens % page, (new_lens // page).clamp(max=table.shape[1] - 1).long()
    rows = torch.arange(N, device=refs.device)
    page_of = new[rows, last].long()
    cut = part > 0
    here = _how_often(page_of[cut].to(torch.int32), P)  # new rows that would write to a page
    first = torch.full((P,), N, dtype=torch.int64, device=refs.device).scatter_reduce_(0, page_of[cut], rows[cut], "amin")
    at = page_of.clamp(min=0)
    copied = cut & ((refs[at] > here[at]) | (first[at] != rows))
    who = torch.nonzero(copied)[:, 0]
    src, dst = page_of[who], _free_ones(refs)[:who.shape[0]]
    refs -= _how_often(src.to(torch.int32), P)
    refs[dst] = 1
    new[who, last[who]] = dst.to(torch.int32)
    moves = torch.full((3, N), -1, dtype=torch.int32, device=refs.device)
    moves[:, :who.shape[0]] = torch.stack((src, dst, part[who])).to(torch.int32)
    _plain_copy(s["pages"], src, dst, part[who], page)
    return [new, new_lens, moves, refs] + s["pages"]


def _plain_compact(s):
    refs, table, lens, page = s["refs"], s["table"], s["lens"], s["case"]["page"]
    P = refs.shape[0]
    held = refs > 0
    n = int(held.sum())
    numbers = torch.arange(P, device=refs.device)
    src, dst = numbers[held & (numbers >= n)], numbers[~held & (numbers < n)]
    places = torch.where(held, numbers, -1).to(torch.int32)
    places[src] = dst.to(torch.int32)
    _plain_copy(s["pages"], src, dst, None, page)
    table.copy_(torch.where(_pages_held(table, lens, page), places[table.clamp(min=0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0
    moves = torch.full((2, P // 2), -1, dtype=torch.int32, device=refs.device)
    moves[:, :src.shape[0]] = torch.stack((src, dst)).to(torch.int32)
    return [places, moves, table, refs] + s["pages"]


def _plain_turnover(s):
    refs, table, lens, page, gone = s["refs"], s["table"], s["lens"], s["case"]["page"], s["ended"]
    refs -= _how_often(table[gone][_pages_held(table[gone], lens[gone], page)], refs.shape[0])
    table[gone], lens[gone] = -1, 0
    starts = s["starts"]
    before, after = (lens + (page - 1)) // page, (lens + starts[1:] - starts[:-1] + (page - 1)) // page
    rank = torch.cumsum(after - before, 0) - (after - before)
    places = torch.arange(table.shape[1], device=refs.device)
    fresh = (places >= before[:, None]) & (places < after[:, None])
    taken = _free_ones(refs)
    table.copy_(torch.where(fresh, taken[(rank[:, None] + places - before[:, None]).clamp(0, refs.shape[0] - 1)].to(torch.int32), table))
    refs[table[fresh].long()] = 1
    t = torch.arange(s["tokens"], device=refs.device)
    row = torch.searchsorted(starts, t.to(torch.int32), right=True) - 1
    place = lens[row] + t - starts[row]
    slots = table[row, place // page].long() * page + place % page
    lens += starts[1:] - starts[:-1]
    return [slots, table, lens, refs]


def run(state):
    s, op = state, state["case"]["op"]
    if "live" in s:
        s["live"].copy_(s["as_it_was"])
    if own:
        from cachegen_b200 import paged
        page = s["case"]["page"]
        if op == "select":
            return list(paged.beam_select(s["logits"], s["scores"], s["case"]["k"]))
        if op == "copy":
            paged.copy_pages(*s["pages"], s["src"], s["dst"], tokens=s["tokens"])
            return s["pages"]
        if op == "fork":
            return list(paged.fork_pages(s["table"], s["lens"], s["parents"], s["refs"], *s["pages"], release=s["case"]["release"])) + [s["refs"]] + s["pages"]
        if op == "compact":
            return list(paged.compact_pages(s["table"], s["lens"], s["refs"], *s["pages"])) + [s["table"], s["refs"]] + s["pages"]
        paged.free_pages(s["table"], s["lens"], s["refs"], page, rows=s["ended"])
        slots = paged.extend_pages(s["table"], s["lens"], s["refs"], page, q_starts=s["starts"], tokens=s["tokens"])
        return [slots, s["table"], s["lens"], s["refs"]]
    if op == "select":
        return _plain_select(s)
    if op == "copy":
        _plain_copy(s["pages"], s["src"], s["dst"], s["tokens"], s["case"]["page"])
        return s["pages"]
    return {"fork": _plain_fork, "compact": _plain_compact, "turnover": _plain_turnover}[op](s)


def _exact_select(case, s):
    """Request by request on the host: log softmax of each row by its definition, and the best of the candidates in order."""
    B, K, V, k = case["batch"], case["beams"], case["vocab"], case["k"]
    got = np.full((B, k), -np.inf)
    tokens, parents = np.full((B, k), -1, dtype=np.int32), np.full((B, k), -1, dtype=np.int32)
    scores = s["scores"].double().cpu().numpy()
    for b in range(B):
        values, where = [], []
        for i in range(K):
            if scores[b, i] == -np.inf:
                continue
            x = s["logits"][b * K + i].double().cpu().numpy()
            at = np.flatnonzero(x > -np.inf)
            if not at.size:
                continue
            x = x[at]
            top = x.max()
            whole = top + np.log(np.exp(x - top).sum())
            if at.size > k:  # a row's best k, and what equals the last of them
                best = x >= np.partition(x, at.size - k)[at.size - k]
                x, at = x[best], at[best]
            values.append(scores[b, i] + (x - whole))
            where.append(i * V + at)
        if not values:
            continue
        values, where = np.concatenate(values), np.concatenate(where)
        order = np.lexsort((where, -values))[:k]
        n = order.size
        got[b, :n], tokens[b, :n], parents[b, :n] = values[order], where[order] % V, b * K + where[order] // V
    return [torch.from_numpy(t).cuda() for t in (got, tokens, parents)]


def _exact_pages(pages, moves, page):
    """Copies one by one; moves: (from, to, tokens)."""
    out = [t.double() for t in pages]
    for t, o in zip(pages, out):
        for a, b, n in moves:
            o[..., b, :n, :, :] = t[..., a, :n, :, :].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(case, s)
    page = case["page"]
    if case["op"] == "copy":
        tokens = [page] * case["pages"] if s["tokens"] is None else s["tokens"].tolist()
        return _exact_pages(s["pages"], list(zip(s["src"].tolist(), s["dst"].tolist(), tokens)), page)
    refs, table, lens = s["refs"].tolist(), s["table"].tolist(), s["lens"].tolist()

    def back(*what):
        return [torch.tensor(w, dtype=torch.int32, device="cuda") for w in what]

    if case["op"] == "fork":
        parents, width = s["parents"].tolist(), len(table[0])
        new = [table[p][:_need(lens[p], page)] + [-1] * (width - _need(lens[p], page)) for p in parents]
        new_lens = [lens[p] for p in parents]
        for rows, ns, step in ((new, new_lens, 1), (table, lens, -1 if case["release"] else 0)):
            for row, n in zip(rows, ns):
                for p in row[:_need(n, page)]:
                    refs[p] += step
        writers = {}
        for i, n in enumerate(new_lens):
            if n % page:
                writers.setdefault(new[i][n // page], []).append(i)
        mine = {rows[0] for p, rows in writers.items() if refs[p] == len(rows)}
        free, moves = iter([p for p, c in enumerate(refs) if c == 0]), []
        for i, n in enumerate(new_lens):
            if n % page and i not in mine:
                a, b = new[i][n // page], next(free)
                refs[a], refs[b], new[i][n // page] = refs[a] - 1, 1, b
                moves.append((a, b, n % page))
        listed_moves = [[m[c] for m in moves] + [-1] * (len(parents) - len(moves)) for c in range(3)]
        return back(new, new_lens, listed_moves, refs) + _exact_pages(s["pages"], moves, page)
    if case["op"] == "compact":
        n = sum(c > 0 for c in refs)
        holes = iter([p for p in range(n) if refs[p] == 0])
        places, moves = [-1] * len(refs), []
        for p, c in enumerate(refs):
            if c > 0:
                places[p] = p if p < n else next(holes)
                if p >= n:
                    moves.append((p, places[p], page))
        after = [0] * len(refs)
        for p, c in enumerate(refs):
            if c > 0:
                after[places[p]] = c
        for row, m in zip(table, lens):
            row[:_need(m, page)] = [places[p] for p in row[:_need(m, page)]]
        listed_moves = [[m[c] for m in moves] + [-1] * (len(refs) // 2 - len(moves)) for c in range(2)]
        return back(places, listed_moves, table, after) + _exact_pages(s["pages"], moves, page)
    for i in s["ended"].tolist():
        for p in table[i][:_need(lens[i], page)]:
            refs[p] -= 1
        table[i], lens[i] = [-1] * len(table[i]), 0
    starts, slots = s["starts"].tolist(), []
    free = iter([p for p, c in enumerate(refs) if c == 0])
    for i in range(len(lens)):
        for place in range(lens[i], lens[i] + starts[i + 1] - starts[i]):
            if place % page == 0:
                table[i][place // page] = next(free)
                refs[table[i][place // page]] = 1
            slots.append(table[i][place // page] * page + place % page)
        lens[i] += starts[i + 1] - starts[i]
    return [torch.tensor(slots, dtype=torch.int64, device="cuda")] + back(table, lens, refs)
