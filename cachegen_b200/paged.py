"""A paged KV cache: where decoded contexts are used (no counterpart in the reference, whose engine hands blobs on).

    Rotary            frequencies and layout of a model's rotary positions
    apply_rotary      positions put into vectors, or taken out of them
    append_paged      keys and values of new tokens, or a blob of every layer, into pages, rotated on the way
    gather_paged      a range of a cache out of its pages, rotation undone on the way
    paged_attention   attention of the newest tokens of a batch of requests over their pages
    check_status      raises if a kernel met a slot, page or length that does not fit

Pages are tensors [num_pages, page_size, heads, head_size] of float16 or bfloat16, with any strides but an innermost one of 1
(a cache that keeps a head's tokens together is passed as a transposed view); with a leading axis where a call is
made for several layers.  Slot s is token s % page_size of page s // page_size.

Calls enqueue on the current stream of the tensors' device, allocate what they return and a workspace from
torch's allocator, and wait for nothing, so they can be captured in a CUDA graph (which needs its Rotary as long as it is replayed, and
reports to check_status if there was a call in front of its capture).  They compute no gradients.  The kernels
check slots, pages and lengths: what lies outside is left out and noted for check_status.
CacheGenDeserializer.decode_paged and CacheGenSerializer.encode_paged connect pages with the codec.
"""
import ctypes
import math
from fractions import Fraction
from typing import Optional

import torch

from . import _lib
from .serde.cachegen_basics import on_device
from .torchac_cuda import _check, _status, _status_word

_DTYPES = {torch.float16: _lib.CG_F16, torch.bfloat16: _lib.CG_BF16}
_INDEX = (torch.int32, torch.int64)
_TWO_PI = Fraction(628318530717958647692528676655900576839, 10 ** 38)


class Rotary:
    """Rotary positions of vectors of `head_size` values: pair i of the first `rotary_dims` (default: all) turns by
    p * w_i radians at position p, w_i = base ** (-2 i / rotary_dims).  The pair is values (i, i + rotary_dims / 2), or (2i, 2i + 1)
    when `interleaved`.  `scaling` changes the frequencies for contexts longer than a model was trained on:

        ("linear", factor)                     w_i / factor: positions closer together
        ("ntk", factor)                        base * factor ** (r / (r - 2)), r = rotary_dims: fast pairs keep their
                                               speed, the slowest turns factor times slower
        ("bands", factor, low, high, trained)  pairs that turn fewer than `low` times in `trained` positions are slowed by factor,
                                               those with more than `high` turns are left, with a linear ramp in between

    `frequencies` (rotary_dims / 2 numbers, radians a position) replaces all that.  Positions may be any 64-bit integers: angles are
    binary fractions of a turn in 64 bits, off by |p| * 2^-65 turns (and 2^-26 for the cosine's argument), so 2^-25 at 2^40 and 0.0002 radians at 2^50."""

    def __init__(self, head_size: int, base: float = 10000.0, rotary_dims: int = None, interleaved: bool = False,
                 scaling: tuple = None, frequencies=None):
        r = head_size if rotary_dims is None else rotary_dims
        if head_size <= 0 or r <= 0 or r % 2 or r > head_size:
            raise ValueError(f"rotary_dims must be even and between 2 and the head size, got {r} of {head_size}")
        if frequencies is not None:
            if scaling is not None:
                raise ValueError("scaling changes the frequencies of `base`; given ones are used as they are")
            w = [float(f) for f in frequencies]
            if len(w) != r // 2:
                raise ValueError(f"expected {r // 2} frequencies, got {len(w)}")
        else:
            w = _frequencies(r, base, scaling)
        if not all(math.isfinite(f) for f in w):
            raise ValueError("frequencies must be finite")
        self.head_size, self.rotary_dims, self.interleaved = head_size, r, bool(interleaved)
        self.frequencies = tuple(w)
        turns = [_turns(f) for f in w]
        self._turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64)
        self._on, self._made_on = {}, {}  # by device: the turns, and the stream whose memory they have
        if torch.cuda.is_available():
            self.turns(torch.device("cuda", torch.cuda.current_device()))

    def turns(self, device) -> torch.Tensor:
        """2^64ths of a turn a position, on `device`; made when a device is first asked for, which a graph's capture must not be."""
        t = self._on.get(device)
        if t is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a Rotary is used on its device once before a capture there")
            with torch.inference_mode(False):
                t = self._turns.to(device)  # from pageable memory: there for every stream when the call returns
            self._made_on[device] = _stream(device)
            self._on[device] = t
        return t

    def __getstate__(self):  # copies make their own
        return {**self.__dict__, "_on": {}, "_made_on": {}}


def _turns(radians: float) -> int:
    """An angle as 2^64ths of a turn, rounded to nearest, without whole turns.  (In integers: a Fraction takes 4 us.)"""
    num, den = radians.as_integer_ratio()
    d = 2 * den * _TWO_PI.numerator
    return ((num << 65) * _TWO_PI.denominator + d // 2) // d % 2 ** 64


def _frequencies(r: int, base: float, scaling: Optional[tuple]) -> list:
    kind = None if scaling is None else scaling[0]
    sizes = {None: 0, "linear": 2, "ntk": 2, "bands": 5}
    if kind not in sizes or scaling is not None and len(scaling) != sizes[kind]:
        raise ValueError(f"unknown scaling {scaling!r}")
    if base <= 0 or scaling is not None and not all(x > 0 for x in scaling[1:]):
        raise ValueError("base and the numbers of a scaling must be positive")
    if kind == "ntk":
        if r < 4:
            raise ValueError("ntk scaling needs two pairs")
        base = base * scaling[1] ** (r / (r - 2))
    w = [base ** (-2.0 * i / r) for i in range(r // 2)]
    if kind == "linear":
        w = [f / scaling[1] for f in w]
    if kind == "bands":
        _, factor, low, high, trained = scaling
        if high <= low:
            raise ValueError("bands: high must be above low")
        keep = [min(1.0, max(0.0, (trained * f / (2 * math.pi) - low) / (high - low))) for f in w]
        w = [f / factor * (1.0 - k) + f * k for f, k in zip(w, keep)]
    return w


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _rows(t, name, device, dtype, rank, shape, written=False):
    """Checks a tensor of rows; shape: what is known of its sizes (None: any)."""
    _check(t.is_cuda and t.device == device, f"{name} must be on {device}")
    _check(t.dtype == dtype, f"{name} must be {dtype}, as the other tensors of the call")
    _check(t.dim() == rank, f"{name} must have {rank} dimensions")
    _check(all(w is None or n == w for n, w in zip(t.shape, shape)), f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    _check(t.stride(-1) == 1 or t.shape[-1] <= 1, f"{name} must have an innermost stride of 1")
    if written:
        _check(all(s or n <= 1 for s, n in zip(t.stride(), t.shape)), f"{name} is written to and must not be expanded")
    _check(not t.is_neg(), f"{name} is a view that negates its memory")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient, which calls on a paged cache do not compute")


def _indices(t, name, device, shape):
    _check(t.is_cuda and t.device == device, f"{name} must be on {device}")
    _check(t.dtype in _INDEX, f"{name} must be int32 or int64")
    _check(tuple(t.shape) == shape, f"{name} has shape {tuple(t.shape)}, expected {shape}")
    _check(t.is_contiguous(), f"{name} must be contiguous")
    _check(not t.is_neg(), f"{name} is a view that negates its memory")


def _head(t, name):
    _check(t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.dtype in _DTYPES, f"{name} must be float16 or bfloat16, got {t.dtype}")
    _check(t.dim() in (3, 4), f"{name} must have shape [tokens, heads, head_size], with a leading axis for several layers")


def _turning(job, rotary, positions, device, shape, D):
    if rotary is None:
        _check(positions is None, "positions are given, but no rotary")
        return
    _check(positions is not None, "rotary needs the tokens' positions")
    _check(rotary.head_size == D, f"rotary is for heads of {rotary.head_size} values, these have {D}")
    if positions.dim() == 2 and len(shape) == 2:
        _indices(positions, "positions", device, shape)
        job.pos_layer = shape[1] if shape[0] > 1 else 0
    else:
        _indices(positions, "positions", device, shape[-1:])
    job.positions, job.wide_positions = positions.data_ptr(), positions.dtype == torch.int64
    turns = rotary.turns(device)
    if not torch.cuda.is_current_stream_capturing():
        turns.record_stream(torch.cuda.current_stream(device))  # a Rotary may be dropped while the kernel reads them
    job.turns = turns.data_ptr()
    job.rotary_dims, job.interleaved = rotary.rotary_dims, rotary.interleaved


def _status_of(t):
    """The status word of a tensor's GPU; None for a tensor on none, and in a capture in front of which there was no call: the word
    outlives the graph, so it must not come from the graph's memory."""
    if not t.is_cuda or (torch.cuda.is_current_stream_capturing() and (t.device.type, t.device.index) not in _status):
        return None
    return _status_word(t.device)


def _set(job, **counts):
    """Fields of a job that are 32-bit counts.  (ctypes cuts a larger number off without a word.)"""
    for name, n in counts.items():
        _check(n < 2 ** 31, f"{name}: {n} is more than a call takes")
        setattr(job, name, n)


def _address(t):
    return None if t is None else t.data_ptr()


def _turns_for(rotary, t):
    """What the native calls take of a Rotary, for tensors on t's GPU."""
    if rotary is None or not t.is_cuda:
        return None, 0, 0, False, 0
    turns = rotary.turns(t.device)
    return turns, rotary._made_on[t.device], rotary.rotary_dims, rotary.interleaved, rotary.head_size


def _finish(done, what):
    """The result of a native call; an error code becomes the error."""
    if type(done) is int:
        _lib.check(done, what)
    return done


def _run(entry, job, device):
    with on_device(device):
        rc = getattr(_lib.lib(), entry)(ctypes.byref(job), _stream(device))
    _lib.check(rc, entry)


def _wrote(*tensors):
    """Tells torch that tensors were written to: a backward pass that kept one for later must not use what is in it now."""
    for t in tensors:
        if t is not None and not t.is_inference():  # (those have no versions)
            torch.autograd.graph.increment_version(t)


def _same_or_apart(a, b, names):
    """Whether a call may read a while it writes b."""
    if a.data_ptr() == b.data_ptr() and a.stride() == b.stride():
        return
    _check(_are_apart(a, b), f"{names} must be the same tensor or not overlap")


def _are_apart(a, b):
    """Whether two tensors of 16-bit values share none: the ranges of memory from the first to the last value do not overlap, or, as
    with the parts of one array, the axes that they step along together (from the widest step on) keep their values apart."""
    if not a.numel() or not b.numel():
        return True
    axes = [sorted(((s, n) for s, n in zip(t.stride(), t.shape) if n > 1), reverse=True) for t in (a, b)]
    return _no_value_shared(b.data_ptr() - a.data_ptr(), *axes)


def _no_value_shared(gap, a, b):
    """The same for what begins `gap` bytes apart and has these (stride, size) axes, the widest strides first."""
    if gap >= 2 * _span(a) or -gap >= 2 * _span(b):
        return True
    step = max(axes[0][0] for axes in (a, b) if axes) if a or b else 0
    if step == 0:
        return False
    (na, rest_a), (nb, rest_b) = ((x[0][1], x[1:]) if x and x[0][0] == step else (1, x) for x in (a, b))
    step, reach_a, reach_b = 2 * step, 2 * _span(rest_a), 2 * _span(rest_b)
    # step i of a and step i - k of b begin gap - k * step apart: those k at which their rests' ranges meet (many only in odd layouts)
    first = max((gap - reach_a) // step + 1, 1 - nb)
    last = min(-((-gap - reach_b) // step) - 1, na - 1)
    return last - first < 4 and all(_no_value_shared(gap - k * step, rest_a, rest_b) for k in range(first, last + 1))


def _span(axes):
    """Values from the first to the last."""
    return 1 + sum((n - 1) * s for s, n in axes)


def apply_rotary(x: torch.Tensor, positions: torch.Tensor, rotary: Rotary, out: torch.Tensor = None,
                 inverse: bool = False) -> torch.Tensor:
    """x [tokens, heads, head_size] or [n, tokens, heads, head_size] with every token turned to its position (`inverse`: back from
    it), in `out` (which may be x) or a new tensor.  positions: int32 or int64 [tokens], or [n, tokens].
    Moving cached keys by d positions is a turn by d: positions of d everywhere."""
    if rotary is not None:
        done = _lib.calls().rotary(x, out, bool(inverse), *_turns_for(rotary, x), positions)
        if done is not None:
            return _finish(done, "apply_rotary")
    _head(x, "x")
    T, H, D = x.shape[-3:]
    dev = x.device
    _rows(x, "x", dev, x.dtype, x.dim(), x.shape)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    else:
        _rows(out, "out", dev, x.dtype, x.dim(), x.shape, written=True)
        _same_or_apart(x, out, "x and out")
    lead = x.shape[0] if x.dim() == 4 else 1
    job = _lib.RowsJob()
    _turning(job, rotary, positions, dev, (lead, T) if x.dim() == 4 else (T,), D)
    _check(rotary is not None, "apply_rotary needs a Rotary")
    job.k, job.k_out = x.data_ptr(), out.data_ptr()
    job.k_strides[:], job.k_out_strides[:] = _dense(x), _dense(out)
    job.dtype, job.inverse = _DTYPES[x.dtype], bool(inverse)
    _set(job, nlayers=lead, ntokens=T, heads=H, head_size=D)
    _run("cg_rotary", job, dev)
    _wrote(out)
    return out


def _dense(t):
    """{layer, token, head} strides of rows."""
    s = t.stride()
    return s[:3] if len(s) == 4 else (0, s[0], s[1])


def _paged(t):
    """{layer, page, token, head} strides of pages."""
    s = t.stride()
    return s[:4] if len(s) == 5 else (0, s[0], s[1], s[2])


def _pages_job(k, v, k_pages, v_pages, slots, rotary, positions, written):
    """What append_paged and gather_paged have in common; `written`: whether the pages are what is written."""
    lead, (T, H, D) = tuple(k.shape[:-3]), k.shape[-3:]
    dev, dtype, rank = k.device, k.dtype, k.dim()
    _rows(k, "k", dev, dtype, rank, k.shape, not written)
    _rows(v, "v", dev, dtype, rank, k.shape, not written)
    _check(k_pages.dim() == rank + 1, f"k_pages must have {rank + 1} dimensions, as k has {rank}")
    P, S = k_pages.shape[-4:-2]
    _rows(k_pages, "k_pages", dev, dtype, rank + 1, lead + (P, S, H, D), written)
    _rows(v_pages, "v_pages", dev, dtype, rank + 1, lead + (P, S, H, D), written)
    written_k, written_v, names = (k_pages, v_pages, "k_pages and v_pages") if written else (k, v, "k and v")
    _check(not T or written_k.data_ptr() != written_v.data_ptr(), f"{names} must not be the same memory")
    if T:
        _check(_are_apart(written_k, written_v), f"{names} must not overlap")
    _indices(slots, "slots", dev, (T,))
    job = _lib.RowsJob()
    _turning(job, rotary, positions, dev, (T,), D)
    job.k, job.v, job.pages_k, job.pages_v = k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    job.k_strides[:], job.v_strides[:] = _dense(k), _dense(v)
    job.pages_k_strides[:], job.pages_v_strides[:] = _paged(k_pages), _paged(v_pages)
    job.slots, job.wide_slots, job.status = slots.data_ptr(), slots.dtype == torch.int64, _address(_status_of(k))
    job.dtype, job.num_pages = _DTYPES[dtype], P if S else 0
    _set(job, nlayers=lead[0] if lead else 1, ntokens=T, heads=H, head_size=D, page_size=max(S, 1))
    return job


def append_paged(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor,
                 rotary: Rotary = None, positions: torch.Tensor = None, q: torch.Tensor = None,
                 q_out: torch.Tensor = None) -> Optional[torch.Tensor]:
    """Writes k and v [tokens, heads, head_size] to the slots (int32 or int64 [tokens]) of their tokens; with a leading axis of
    layers, to the same slots of every layer's pages.  With `rotary` the keys, and the queries q [tokens, q_heads, head_size] if
    there are any, are turned to `positions` [tokens] on the way.  Returns the queries: q_out (which may be q, nothing else) or a new
    tensor.  A token with slot -1 is padding: nothing of it is written, its row of q_out neither.  Each slot belongs to one token:
    of two that name the same, either may be found there, or pieces of both."""
    done = _lib.calls().append(k, v, k_pages, v_pages, slots, _status_of(k), *_turns_for(rotary, k), positions, q, q_out)
    if done is not None:
        done = _finish(done, "append_paged")
        return None if done is True else done
    _head(k, "k")
    job = _pages_job(k, v, k_pages, v_pages, slots, rotary, positions, True)
    for name, t in (("k", k), ("v", v)):
        for other, pages in (("k_pages", k_pages), ("v_pages", v_pages)):
            _apart(t, pages, name, other)
    if q is None:
        _check(q_out is None, "q_out is given, but no q")
    else:
        _check(k.dim() == 3, "queries are rotated beside the keys of one layer")
        _rows(q, "q", k.device, k.dtype, 3, (k.shape[0], None, k.shape[2]))
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            _rows(q_out, "q_out", k.device, k.dtype, 3, q.shape, written=True)
            _same_or_apart(q, q_out, "q and q_out")
            for name, t in (("k", k), ("v", v), ("k_pages", k_pages), ("v_pages", v_pages)):
                _apart(q_out, t, "q_out", name)
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            _apart(q, t, "q", name)
        job.q, job.q_out = q.data_ptr(), q_out.data_ptr()
        _set(job, q_heads=q.shape[1])
        job.q_strides[:], job.q_out_strides[:] = _dense(q), _dense(q_out)
    _run("cg_append_paged", job, k.device)
    _wrote(k_pages, v_pages, q_out)
    return q_out


def gather_paged(k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor, k: torch.Tensor = None,
                 v: torch.Tensor = None, rotary: Rotary = None, positions: torch.Tensor = None) -> tuple:
    """The keys and values of the slots (int32 or int64 [tokens]), as k and v [tokens, heads, head_size] (new tensors if not given);
    of all layers if the pages have a leading axis.  With `rotary` the keys are turned back from `positions` [tokens].  Rows of
    tokens with slot -1 are left as they are."""
    done = _lib.calls().gather(k, v, k_pages, v_pages, slots, _status_of(k_pages), *_turns_for(rotary, k_pages), positions)
    if done is not None:
        return _finish(done, "gather_paged")
    _check(k_pages.is_cuda, "k_pages must be a CUDA tensor")
    _check(k_pages.dtype in _DTYPES, f"k_pages must be float16 or bfloat16, got {k_pages.dtype}")
    _check(k_pages.dim() in (4, 5), "k_pages must have shape [pages, page_size, heads, head_size], with a leading axis for several layers")
    _check(slots.dim() == 1, "slots must have one dimension")
    shape = tuple(k_pages.shape[:-4]) + (slots.shape[0],) + tuple(k_pages.shape[-2:])
    k = torch.empty(shape, dtype=k_pages.dtype, device=k_pages.device) if k is None else k
    v = torch.empty(shape, dtype=k_pages.dtype, device=k_pages.device) if v is None else v
    _check(tuple(k.shape) == shape, f"k has shape {tuple(k.shape)}, expected {shape}")
    _check(k.is_cuda and k.dtype in _DTYPES, "k must be a float16 or bfloat16 CUDA tensor")
    job = _pages_job(k, v, k_pages, v_pages, slots, rotary, positions, False)
    for name, t in (("k", k), ("v", v)):
        for other, pages in (("k_pages", k_pages), ("v_pages", v_pages)):
            _apart(t, pages, name, other)
    _run("cg_gather_paged", job, k.device)
    _wrote(k, v)
    return k, v


def _apart(a, b, name_a, name_b):
    _check(_are_apart(a, b), f"{name_a} must not overlap {name_b}")


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                    q_starts: torch.Tensor = None, scale: float = None, causal: bool = True, window: int = 0, max_q: int = 0,
                    out: torch.Tensor = None, return_lse: bool = False):
    """Attention of the newest tokens of a batch of requests over their pages.

    q [rows, q_heads, head_size]: rows q_starts[b] .. q_starts[b + 1] - 1 (int32 [requests + 1]; None: one row a request) are the newest
    tokens of request b, whose kv_lens[b] (int32) tokens, the newest included, lie in the pages page_table[b] (int32 [requests, width],
    in order; what stands behind the last page that a request needs is not read).  q_heads is a multiple of the cache's heads; query
    head h reads head h // (q_heads // heads).  Row i of n, at place p = kv_len - n + i, sees the keys up to its own place (all
    keys if not `causal`), with window > 0 only those behind p - window.  A row that sees none gets zeros (and -inf).
    scale: of the scores, 1 / sqrt(head_size) by default.  max_q: the most rows of a request, if the caller knows; without it
    all rows may be one request's, and single tokens of many requests then take longer than they need.

    Returns `out` (a new tensor if not given; rows of no request are left as they are), with return_lse also the float32
    logarithm of each row's sum of exponentials [rows, q_heads]."""
    scale = 1.0 / math.sqrt(max(q.shape[-1], 1)) if scale is None else float(scale)
    causal, return_lse = bool(causal), bool(return_lse)
    done = _lib.calls().attend(q, k_pages, v_pages, page_table, kv_lens, q_starts, scale, causal, window, max_q, out, return_lse, _status_of(q))
    if done is not None:
        return _finish(done, "paged_attention")
    _check(q.is_cuda, "q must be a CUDA tensor")
    _check(q.dtype in _DTYPES, f"q must be float16 or bfloat16, got {q.dtype}")
    dev, dtype = q.device, q.dtype
    _rows(q, "q", dev, dtype, 3, (None, None, None))
    R, Q, D = q.shape
    _check(k_pages.dim() == 4, "k_pages must have 4 dimensions")
    P, S, H, _ = k_pages.shape
    _rows(k_pages, "k_pages", dev, dtype, 4, (P, S, H, D))
    _rows(v_pages, "v_pages", dev, dtype, 4, (P, S, H, D))
    _check(D % 8 == 0 and 0 < D <= 128, f"head_size must be a multiple of 8 up to 128, got {D}")
    _check(S > 0, "pages must hold a token at least")
    _check(H > 0 and Q > 0 and Q % H == 0, f"{Q} query heads cannot share {H} heads of the cache")
    B = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    _check(B >= 0, "kv_lens must have one dimension")
    _check(B <= _lib.CG_MAX_REQUESTS, f"at most {_lib.CG_MAX_REQUESTS} requests in a call")
    for name, t, shape in (("kv_lens", kv_lens, (B,)), ("page_table", page_table, (B, None)), ("q_starts", q_starts, (B + 1,))):
        if t is None:
            continue
        _check(t.is_cuda and t.device == dev, f"{name} must be on {dev}")
        _check(t.dtype == torch.int32, f"{name} must be int32")
        _check(not t.is_neg(), f"{name} is a view that negates its memory")
        _check(t.dim() == len(shape) and all(w in (None, n) for w, n in zip(shape, t.shape)), f"{name} has shape {tuple(t.shape)}, expected {shape}")
        _check(t.stride(-1) == 1 or t.shape[-1] <= 1, f"{name} must have an innermost stride of 1")
    _check(q_starts is not None or R == B, f"without q_starts each of {B} requests has one row, q has {R}")
    _check(window >= 0 and max_q >= 0, "window and max_q must not be negative")
    if out is None:
        out = torch.empty((R, Q, D), dtype=dtype, device=dev)
    else:
        _rows(out, "out", dev, dtype, 3, q.shape, written=True)
        for name, t in (("q", q), ("k_pages", k_pages), ("v_pages", v_pages)):
            _apart(out, t, "out", name)
    for name, t in (("q", q), ("k_pages", k_pages), ("v_pages", v_pages), ("out", out)):
        _check(t.data_ptr() % 16 == 0 and all(s % 8 == 0 or n <= 1 for s, n in zip(t.stride()[:-1], t.shape)),
               f"{name} must start at a multiple of 16 bytes, with strides that are multiples of 8 values")
    lse = torch.empty((R, Q), dtype=torch.float32, device=dev) if return_lse else None
    job = _lib.AttentionJob()
    job.q, job.pages_k, job.pages_v, job.out = q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr()
    job.lse = lse.data_ptr() if return_lse else None
    job.table, job.kv_lens, job.status = page_table.data_ptr(), kv_lens.data_ptr(), _address(_status_of(q))
    job.q_starts = q_starts.data_ptr() if q_starts is not None else None
    job.table_row, job.num_pages = page_table.stride(0), P
    job.q_strides[:], job.out_strides[:] = _steps(q), _steps(out)
    job.pages_k_strides[:], job.pages_v_strides[:] = _steps(k_pages), _steps(v_pages)
    job.dtype, job.causal, job.window, job.max_q, job.scale = _DTYPES[dtype], causal, min(window, 2 ** 31 - 1), min(max_q, 2 ** 31 - 1), scale
    _set(job, nrequests=B, nrows=R, q_heads=Q, heads=H, head_size=D, page_size=S, table_width=page_table.shape[1])
    with on_device(dev):
        need = _lib.lib().cg_paged_attention_workspace(ctypes.byref(job))
        _lib.check(min(need, 0), "paged_attention")
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)  # of the graph's own memory in a capture
            job.workspace, job.workspace_bytes = workspace.data_ptr(), need
        _lib.check(_lib.lib().cg_paged_attention(ctypes.byref(job), _stream(dev)), "paged_attention")
    _wrote(out)
    return (out, lse) if return_lse else out


def _steps(t):
    """Strides of the outer axes, with none for an axis of one."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)]


def split_pages(pages: torch.Tensor, fmt: str) -> tuple:
    """Keys and values of a cache of all layers, as the calls above take them: [layers, 2, pages, page_size, heads, head_size] ("vllm")
    or [layers, 2, pages, heads, page_size, head_size] ("huggingface")."""
    _check(pages.dim() == 6 and pages.shape[1] == 2, "pages must have shape [layers, 2, pages, ...] with six dimensions")
    if fmt == "huggingface":
        pages = pages.transpose(3, 4)
    return pages[:, 0], pages[:, 1]


def split_blob(kv: torch.Tensor, fmt: str) -> tuple:
    """Keys and values [layers, tokens, heads, head_size] of a KV blob: [layers, 2, tokens, heads, head_size] ("vllm") or
    [layers, 2, heads, tokens, head_size] ("huggingface")."""
    if fmt == "huggingface":
        kv = kv.transpose(2, 3)
    return kv[:, 0], kv[:, 1]


def check_status(device=None) -> None:
    """Synchronises and raises if a kernel met a slot, page or length that does not fit since the last check (the
    status word is that of cachegen_b200.torchac_cuda.check_status)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    w = _status_word(device)
    bits = int(w.item())
    if bits:
        w.zero_()
        raise RuntimeError("paged cache: " + _lib.status_text(bits))
