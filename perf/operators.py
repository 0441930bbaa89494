"""Work on a paged KV cache, as measurable cases: where a context that was loaded from a store is used.

A case is one call of a public entry point of cachegen_b200.paged:

    rotary    apply_rotary    positions put into vectors, or the keys of a whole blob moved to other positions
    append    append_paged    keys and values of new tokens, or a decoded blob of every layer, written to a paged cache,
                              keys (and the queries beside them) rotated on the way
    gather    gather_paged    a range of a paged cache taken out as the blob that a serializer reads, rotation undone or not
    attend    paged_attention attention of the newest tokens of a batch of requests over their pages

    dtype            float16 or bfloat16
    layers           0: one layer's tensors without a layer axis
    tokens           rows of the call (rotary, append, gather)
    q_heads, heads   query heads (0: no queries) and key/value heads
    head             values of a head
    rot              rotated values of a head (0: none are rotated); interleaved: pairs (2i, 2i+1), else (i, i + rot/2)
    base, scaling    frequencies: "none", "linear", "ntk" or "bands", for contexts eight times as long
    page             tokens of a page; far: the first position
    batch, chunk, context, ragged    attend: requests, new tokens of the longest, cache of the longest, and how far the
                                     others may fall short of these (a share); window: tokens that a query sees, 0 all

The plain forms here are elementary torch operations in 32 bits (angles in 64), rounded once at the end.
"""
import math

import torch

own = False  # False: the plain forms; True: the calls of cachegen_b200.paged

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
_FACTOR, _LOW, _HIGH, _ORIGINAL = 8.0, 1.0, 4.0, 8192  # of the scaled frequencies


def _case(name, op, **given):
    case = {"op": op, "dtype": "bfloat16", "layers": 0, "tokens": 1, "q_heads": 0, "heads": 8, "head": 128, "rot": 0,
            "interleaved": False, "base": 10000.0, "scaling": "none", "page": 16, "far": 0, "batch": 1, "chunk": 1,
            "context": 1, "ragged": 0.0, "window": 0, "lse": False}
    case.update(given)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one step of eight requests: a call whose time is its launch
        _case("rotary_step_8", "rotary", tokens=8, heads=32, rot=128, far=4000),
        # the keys of a cached context of all layers, moved to where the context stands in another prompt
        _case("rotary_blob_1999", "rotary", layers=32, tokens=1999, rot=128, dtype="float16", scaling="ntk", far=20000),
        # one step of 64 requests: queries and keys rotated, keys and values to their pages
        _case("append_step_64", "append", tokens=64, q_heads=32, heads=8, rot=128, far=3000),
        # a prompt of a multi-head model with half of each head rotated, in neighbouring pairs
        _case("append_prompt_1999", "append", tokens=1999, q_heads=32, heads=32, rot=64, interleaved=True, dtype="float16", page=64),
        # a decoded context of every layer to the pages of a request
        _case("append_blob_8192", "append", layers=32, tokens=8192, heads=8, rot=128, base=500000.0, scaling="bands", far=100000),
        # what a serializer takes of a cache at a time, as it stands
        _case("gather_chunk_256", "gather", layers=32, tokens=256, heads=32, dtype="float16"),
        # a context of a large model, its keys without their positions
        _case("gather_blob_4096", "gather", layers=80, tokens=4096, heads=8, rot=128, page=64),
        # the first step of a short request: latency
        _case("attend_step_61", "attend", q_heads=32, heads=8, context=61),
        # a step of 64 requests of up to 4,096 tokens
        _case("attend_step_64x4096", "attend", q_heads=32, heads=8, batch=64, context=4096, ragged=0.6),
        # a step of one request with a long context
        _case("attend_step_32768", "attend", q_heads=32, heads=8, context=32768, page=64, lse=True),
        # a question of 256 tokens over a loaded context of a large model
        _case("attend_chunk_16384", "attend", q_heads=64, heads=8, chunk=256, context=16384, dtype="float16"),
        # a whole prompt of a multi-head model
        _case("attend_prompt_8192", "attend", q_heads=32, heads=32, chunk=8192, context=8192, page=128),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


_MOST = {"rotary": 1 << 28, "append": 1 << 30, "gather": 1 << 30, "attend": 1 << 30}  # bytes of a drawn case
_MOST_FLOPS = 5e11


def draw(rng):
    op = rng.choice(["rotary", "append", "append", "gather", "attend", "attend", "attend"])
    q_heads, heads = rng.choice([(32, 32), (32, 8), (64, 8), (28, 4), (8, 1), (12, 12)])
    head = rng.choice([128, 128, 128, 64, 80, 96])
    case = _case(None, op, dtype=rng.choice(sorted(_DTYPES)), q_heads=q_heads, heads=heads, head=head,
                 page=rng.choice([16, 16, 64, 32, 128, 8, 1, 24]))
    if op != "attend":
        case["layers"] = rng.choice([0, 0, 1, 10, 32, 80])
        case["tokens"] = _log(rng, 1, 16384)
        case["rot"] = rng.choice([head, head, head // 2, 0 if op != "rotary" else head])
        case["interleaved"] = rng.random() < 0.4
        case["base"] = rng.choice([10000.0, 500000.0])
        case["scaling"] = rng.choice(["none", "linear", "ntk", "bands"])
        case["far"] = rng.choice([0, _log(rng, 1, 1000000)])
        if op != "append" or case["layers"]:
            case["q_heads"] = 0
        while work(case)["bytes"] > _MOST[op]:
            case["tokens"] = case["tokens"] // 2 + 1
        return case
    case["batch"] = _log(rng, 1, 64)
    case["context"] = _log(rng, 1, 32768)
    kind = rng.choice(["step", "step", "chunk", "chunk", "prompt"])
    case["chunk"] = {"step": 1, "chunk": min(case["context"], _log(rng, 2, 1024)), "prompt": case["context"]}[kind]
    case["ragged"] = rng.choice([0.0, 0.3, 0.9])
    case["window"] = rng.choice([0, 0, 0, _log(rng, 1, 8192)])
    case["lse"] = rng.random() < 0.3
    while work(case)["bytes"] > _MOST[op] or work(case)["flops"] > _MOST_FLOPS:
        if case["batch"] > 1:
            case["batch"] = case["batch"] // 2
        else:
            case["context"] = case["context"] // 2 + 1
            case["chunk"] = min(case["chunk"], case["context"])
    return case


def _lengths(case):
    """New tokens and whole length of every request: the first is the longest, the others fall short by up to `ragged`."""
    out = []
    for i in range(case["batch"]):
        short, fewer = ((i * 0.6180339887 + s) % 1.0 * case["ragged"] if i else 0.0 for s in (0.0, 0.37))
        n = max(1, int(case["chunk"] * (1.0 - fewer)))
        out.append((n, max(n, int(case["context"] * (1.0 - short)))))
    return out


def _visible(n, kv, window):
    """Query-key pairs of a request: the i-th of n new tokens sees the keys up to its own, the last `window` of them."""
    first = kv - n + 1
    if not window or window >= kv:
        return n * first + n * (n - 1) // 2
    return sum(min(window, first + i) for i in range(n))


def work(case):
    D, H, Q = case["head"], case["heads"], case["q_heads"]
    if case["op"] == "attend":
        lens = _lengths(case)
        new, pairs = sum(n for n, _ in lens), sum(_visible(n, kv, case["window"]) for n, kv in lens)
        seen = sum(min(kv, n - 1 + case["window"]) if case["window"] else kv for n, kv in lens)
        return {"bytes": 2 * D * (2 * new * Q + 2 * seen * H) + (4 * new * Q if case["lse"] else 0), "flops": 4 * D * Q * pairs}
    rows = max(1, case["layers"]) * case["tokens"]
    if case["op"] == "rotary":
        return {"bytes": 2 * 2 * rows * H * D + 8 * case["tokens"], "flops": 3 * rows * H * case["rot"]}
    turned = H + Q if case["op"] == "append" else H
    return {"bytes": 2 * 2 * rows * D * (2 * H + Q) + 16 * case["tokens"], "flops": 3 * rows * turned * case["rot"]}


def _frequencies(case):
    """Radians a position of every pair, in 64 bits."""
    r, base = case["rot"], case["base"]
    if case["scaling"] == "ntk":  # a larger base: the slowest pair turns as if positions were _FACTOR times closer
        base = base * _FACTOR ** (r / (r - 2))
    w = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if case["scaling"] == "linear":
        w = w / _FACTOR
    if case["scaling"] == "bands":  # slow pairs slowed down, fast ones left, a ramp over their turns in between
        turns = _ORIGINAL * w / (2 * math.pi)
        keep = ((turns - _LOW) / (_HIGH - _LOW)).clamp(0.0, 1.0)
        w = w / _FACTOR * (1 - keep) + w * keep
    return w


def _scaling(case):
    return {"none": None, "linear": ("linear", _FACTOR), "ntk": ("ntk", _FACTOR),
            "bands": ("bands", _FACTOR, _LOW, _HIGH, _ORIGINAL)}[case["scaling"]]


def _normal(g, shape, dtype):
    """Values as a model's projections give them: channels of unlike scale, a few ten times larger."""
    scale = torch.exp(0.4 * torch.randn(shape[-2:], generator=g, device="cuda"))
    scale = torch.where(torch.rand(shape[-2:], generator=g, device="cuda") < 0.01, scale * 10.0, scale)
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1, *shape[-2:])
    step = max(1, (1 << 26) // max(1, flat[0].numel()))
    for at in range(0, flat.shape[0], step):
        part = flat[at:at + step]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * scale)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, D, H, Q, page = _DTYPES[case["dtype"]], case["head"], case["heads"], case["q_heads"], case["page"]
    state = {"case": case}
    if own and case["rot"]:
        from cachegen_b200 import paged
        state["rotary"] = paged.Rotary(D, base=case["base"], rotary_dims=case["rot"], interleaved=case["interleaved"],
                                       scaling=_scaling(case))
    if case["op"] == "attend":
        lens = _lengths(case)
        need = [(kv + page - 1) // page for _, kv in lens]
        pool = sum(need) + 3
        order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")  # unused entries name no page
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        state["pages_k"], state["pages_v"] = (_normal(g, (pool, page, H, D), dtype) for _ in range(2))
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        state["q"] = _normal(g, (starts[-1], Q, D), dtype)
        state["table"] = table
        state["kv_lens"] = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
        state["q_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        state["max_q"] = case["chunk"]  # a scheduler knows the longest chunk of its batch
        return state
    T = case["tokens"]
    lead = (case["layers"],) if case["layers"] else ()
    state["positions"] = torch.arange(case["far"], case["far"] + T, device="cuda")
    if case["op"] == "rotary":
        state["x"] = _normal(g, lead + (T, H, D), dtype)
        state["out"] = torch.empty_like(state["x"])
        return state
    pool = (T + page - 1) // page + 3
    order = torch.randperm(pool, generator=g, device="cuda")
    at = torch.arange(T, device="cuda")
    state["slots"] = order[at // page] * page + at % page
    state["pages_k"], state["pages_v"] = (_normal(g, lead + (pool, page, H, D), dtype) for _ in range(2))
    if case["op"] == "append":
        state["k"], state["v"] = (_normal(g, lead + (T, H, D), dtype) for _ in range(2))
        if Q:
            state["q"] = _normal(g, (T, Q, D), dtype)
            state["q_out"] = torch.empty_like(state["q"])
    else:
        # a serializer's blob is one tensor: keys and values are parts of it
        blob = torch.empty(lead + (2, T, H, D), dtype=dtype, device="cuda")
        state["k"], state["v"] = blob.unbind(-4)
    return state


def _turned(x, positions, case, direction):
    """x [..., tokens, heads, head] rotated by its positions (direction 1), or back (-1), in 32 bits."""
    r = case["rot"]
    x = x.float()
    if not r:
        return x
    angle = positions.double()[:, None] * _frequencies(case).to(x.device)
    cos, sin = torch.cos(angle).float()[:, None, :], direction * torch.sin(angle).float()[:, None, :]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        both = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        both = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((both, x[..., r:]), dim=-1)


def _rows(pages):
    """pages [..., pages, page, heads, head] as [..., slots, heads, head]."""
    return pages.flatten(-4, -3)


def _plain_attend(s):
    case, q, out = s["case"], s["q"], torch.zeros_like(s["q"])
    Q, H, D, page = case["q_heads"], case["heads"], case["head"], case["page"]
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float32, device=q.device)
    at, group = 0, Q // H
    for i, (n, kv) in enumerate(_lengths(case)):
        j = torch.arange(kv, device=q.device)
        slots = s["table"][i][j // page].long() * page + j % page
        k, v = _rows(s["pages_k"])[slots].float(), _rows(s["pages_v"])[slots].float()
        own_place = torch.arange(kv - n, kv, device=q.device)[:, None]
        hidden = j > own_place
        if case["window"]:
            hidden = hidden | (j <= own_place - case["window"])
        for h in range(H):
            mine = q[at:at + n, h * group:(h + 1) * group].float().transpose(0, 1) * (1.0 / math.sqrt(D))
            score = (mine @ k[:, h].T).masked_fill(hidden, -math.inf)
            top = score.amax(-1, keepdim=True)
            p = torch.exp(score - top)
            total = p.sum(-1, keepdim=True)
            out[at:at + n, h * group:(h + 1) * group] = (p @ v[:, h] / total).transpose(0, 1).to(out.dtype)
            lse[at:at + n, h * group:(h + 1) * group] = (top + torch.log(total))[..., 0].T
        at += n
    return [out, lse] if case["lse"] else [out]


def run(state):
    s, case = state, state["case"]
    if own:
        from cachegen_b200 import paged
        rotary = s.get("rotary")
        if case["op"] == "rotary":
            return paged.apply_rotary(s["x"], s["positions"], rotary, out=s["out"])
        if case["op"] == "append":
            paged.append_paged(s["k"], s["v"], s["pages_k"], s["pages_v"], s["slots"], rotary=rotary,
                               positions=s["positions"] if rotary else None, q=s.get("q"), q_out=s.get("q_out"))
            return [s["pages_k"], s["pages_v"]] + ([s["q_out"]] if case["q_heads"] else [])
        if case["op"] == "gather":
            paged.gather_paged(s["pages_k"], s["pages_v"], s["slots"], k=s["k"], v=s["v"], rotary=rotary,
                               positions=s["positions"] if rotary else None)
            return [s["k"], s["v"]]
        got = paged.paged_attention(s["q"], s["pages_k"], s["pages_v"], s["table"], s["kv_lens"], s["q_starts"],
                                    window=case["window"], max_q=s["max_q"], return_lse=case["lse"])
        return list(got) if case["lse"] else [got]
    if case["op"] == "rotary":
        s["out"].copy_(_turned(s["x"], s["positions"], case, 1))
        return s["out"]
    if case["op"] == "append":
        _rows(s["pages_k"])[..., s["slots"], :, :] = _turned(s["k"], s["positions"], case, 1).to(s["k"].dtype)
        _rows(s["pages_v"])[..., s["slots"], :, :] = s["v"]
        if not case["q_heads"]:
            return [s["pages_k"], s["pages_v"]]
        s["q_out"].copy_(_turned(s["q"], s["positions"], case, 1))
        return [s["pages_k"], s["pages_v"], s["q_out"]]
    if case["op"] == "gather":
        s["k"].copy_(_turned(_rows(s["pages_k"])[..., s["slots"], :, :], s["positions"], case, -1))
        s["v"].copy_(_rows(s["pages_v"])[..., s["slots"], :, :])
        return [s["k"], s["v"]]
    return _plain_attend(s)


def _exact_turn(x, positions, case, direction):
    """The rotation as a product of complex numbers, in 64 bits."""
    r = case["rot"]
    x = x.double()
    if not r:
        return x
    phase = torch.outer(positions.double(), direction * _frequencies(case).to(x.device))[:, None, :]
    unit = torch.polar(torch.ones_like(phase), phase)
    index = torch.arange(r, device=x.device)
    index = index.view(-1, 2).T if case["interleaved"] else index.view(2, -1)
    z = torch.complex(x[..., index[0]], x[..., index[1]]) * unit
    x[..., index[0]], x[..., index[1]] = z.real, z.imag
    return x


def _exact_attend(case, s):
    """out_i = sum_j exp(q_i k_j / sqrt(D)) v_j / sum_j exp(q_i k_j / sqrt(D)) over the keys that i sees, a block of queries
    of one head at a time."""
    q, D, page, group = s["q"], case["head"], case["page"], case["q_heads"] // case["heads"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    table, row = s["table"].cpu(), 0
    for i, (n, kv) in enumerate(_lengths(case)):
        need = (kv + page - 1) // page
        pages = table[i, :need].long().to(q.device)
        keys, values = (t[pages].reshape(need * page, case["heads"], D)[:kv] for t in (s["pages_k"], s["pages_v"]))
        for head in range(case["heads"]):
            k, v = keys[:, head].double(), values[:, head].double()
            for first in range(0, n, 512):
                count = min(512, n - first)
                see = kv - n + first + count  # no query of the block sees a key behind this
                x = q[row + first:row + first + count, head * group:(head + 1) * group].double()
                score = torch.einsum("ngd,kd->ngk", x, k[:see]) / math.sqrt(D)
                place = torch.arange(kv - n + first, see, device=q.device).view(-1, 1, 1)
                key = torch.arange(see, device=q.device).view(1, 1, -1)
                seen = key <= place
                if case["window"]:
                    seen = seen & (place - key < case["window"])
                score = torch.where(seen, score, torch.full((), -math.inf, dtype=torch.float64, device=q.device))
                whole = torch.logsumexp(score, dim=-1)
                lse[row + first:row + first + count, head * group:(head + 1) * group] = whole
                out[row + first:row + first + count, head * group:(head + 1) * group] = torch.einsum(
                    "ngk,kd->ngd", torch.exp(score - whole[..., None]), v[:see])
        row += n
    return [out, lse] if case["lse"] else [out]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_turn(s["x"], s["positions"], case, 1)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    page, slots = case["page"], s["slots"]
    if case["op"] == "append":
        k, v = s["pages_k"].double(), s["pages_v"].double()
        k[..., slots // page, slots % page, :, :] = _exact_turn(s["k"], s["positions"], case, 1)
        v[..., slots // page, slots % page, :, :] = s["v"].double()
        return [k, v] + ([_exact_turn(s["q"], s["positions"], case, 1)] if case["q_heads"] else [])
    k, v = (t[..., slots // page, slots % page, :, :] for t in (s["pages_k"], s["pages_v"]))
    return [_exact_turn(k, s["positions"], case, -1), v.double()]
