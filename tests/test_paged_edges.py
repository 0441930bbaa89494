"""What the Python path of the calls on a paged cache checks, on tensors that only say that they are on a GPU: nothing is launched."""
import random

import pytest
import torch

from cachegen_b200 import _lib, paged


class OnGpu(torch.Tensor):
    is_cuda = True


def on_gpu(t):
    return t.as_subclass(OnGpu)


@pytest.fixture
def launched(monkeypatch):
    """The names of the calls that would have been launched."""
    names = []
    monkeypatch.setattr(paged, "_run", lambda entry, job, device: names.append(entry))
    monkeypatch.setattr(paged, "_status_of", lambda t: None)
    return names


def values(t):
    """Where a tensor's values lie."""
    at = torch.full((1,), t.data_ptr() // 2)
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n) * s).flatten()
    return set(at.tolist())


def test_tensors_that_share_a_value_are_never_taken_for_apart():
    rng = random.Random(7)
    buffer = torch.zeros(4000, dtype=torch.float16)
    known = 0
    for _ in range(4000):
        views = []
        # parts of one array, by slices and steps of its axes, and any strides at all
        shape = [rng.randint(1, 5) for _ in range(rng.randint(2, 5))]
        array = buffer[:torch.Size(shape).numel()].view(shape).permute(rng.sample(range(len(shape)), len(shape)))
        for _ in range(2):
            if rng.random() < 0.8:
                v = array
                for d in range(v.dim()):
                    first = rng.randrange(v.shape[d])
                    v = v.narrow(d, first, rng.randint(1, v.shape[d] - first))
                    v = v[(slice(None),) * d + (slice(None, None, rng.randint(1, 2)),)]
            else:
                dims = rng.randint(1, 4)
                v = buffer.as_strided([rng.randint(1, 4) for _ in range(dims)], [rng.randint(0, 40) for _ in range(dims)], rng.randint(0, 200))
            views.append(v)
        a, b = views
        apart, shared = paged._are_apart(a, b), bool(values(a) & values(b))
        assert paged._are_apart(b, a) == apart
        assert not (apart and shared)
        known += apart and not shared
    assert known > 1000


def test_parts_of_one_array_are_apart():
    qkv = torch.zeros((9, 12, 64), dtype=torch.float16)  # tokens of queries, keys and values side by side
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    flat = torch.zeros((9, 12 * 64), dtype=torch.float16)
    other = torch.zeros((3, 2, 5, 4, 2, 64), dtype=torch.float16)  # layers, keys and values
    for a, b in ((q, k), (k, v), (q, v), (flat[:, :512], flat[:, 512:640]), (flat[:1, :512], flat[1:2, :512]), (other[:, 0], other[:, 1]),
                 (other[:, 0].transpose(2, 3), other[:, 1].transpose(2, 3)), (other[1, 0], other[1, 1]), (other[:, :, 0], other[:, :, 3]),
                 (other[..., :32], other[..., 32:]), (other[..., 0, :], other[..., 1, :]), (qkv[::2], qkv[1::2]), (q, torch.zeros_like(q)), (q[:0], q)):
        assert paged._are_apart(a, b) and paged._are_apart(b, a)
        assert not a.numel() or not paged._are_apart(a, a)
    for a, b in ((q, qkv[:, 7:9]), (qkv[1:], qkv[:-1]), (other[:, 0], other[:, :, 0]), (flat[:, :513], flat[:, 512:])):
        assert not paged._are_apart(a, b) and not paged._are_apart(b, a)


def rows(*shape):
    return on_gpu(torch.zeros(shape, dtype=torch.float16))


def test_append_and_gather_refuse_what_they_would_read_and_write_at_once(launched):
    """Blocks write some tokens' rows while others read theirs."""
    k, v, q = rows(6, 2, 64), rows(6, 2, 64), rows(6, 2, 64)
    both = rows(2, 3, 4, 2, 64)
    k_pages, v_pages, slots = both[0], both[1], on_gpu(torch.arange(6))
    for q_out in (k, v, k_pages.view(12, 2, 64)[:6], v_pages.view(12, 2, 64)[6:]):
        with pytest.raises(RuntimeError, match="overlap"):
            paged.append_paged(k, v, k_pages, v_pages, slots, q=q, q_out=q_out)
    with pytest.raises(RuntimeError, match="overlap"):
        paged.append_paged(k, v, k_pages, v_pages, slots, q=k_pages.view(12, 2, 64)[:6])
    with pytest.raises(RuntimeError, match="overlap"):
        paged.append_paged(k, v, both.view(6, 4, 2, 64)[:5], both.view(6, 4, 2, 64)[1:], slots)
    seven = rows(7, 2, 64)
    for k_to, v_to in ((k, k), (seven[:6], seven[1:])):
        with pytest.raises(RuntimeError, match="overlap|same memory"):
            paged.gather_paged(k_pages, v_pages, slots, k=k_to, v=v_to)
    assert not launched
    # the parts of one array go, in place too
    qkv = rows(6, 8, 64)
    pages = rows(3, 4, 2, 2, 64)
    q = qkv[:, :4]
    assert paged.append_paged(qkv[:, 4:6], qkv[:, 6:], pages[:, :, 0], pages[:, :, 1], slots, q=q, q_out=q) is q
    kv = rows(6, 2, 2, 64)
    paged.gather_paged(pages[:, :, 0], pages[:, :, 1], slots, k=kv[:, 0], v=kv[:, 1])
    assert launched == ["cg_append_paged", "cg_gather_paged"]


def test_tensors_that_require_a_gradient_are_not_written_to(launched):
    k, v, q, out = rows(6, 2, 64), rows(6, 2, 64), rows(6, 2, 64), rows(6, 2, 64)
    k_pages, v_pages, slots = rows(3, 4, 2, 64), rows(3, 4, 2, 64), on_gpu(torch.arange(6))
    table, lens = on_gpu(torch.zeros((6, 1), dtype=torch.int32)), on_gpu(torch.ones(6, dtype=torch.int32))
    calls = {"k_pages": lambda: paged.append_paged(k, v, k_pages, v_pages, slots), "v_pages": lambda: paged.append_paged(k, v, k_pages, v_pages, slots),
             "q_out": lambda: paged.append_paged(k, v, k_pages, v_pages, slots, q=q, q_out=out),
             "k": lambda: paged.gather_paged(k_pages, v_pages, slots, k=k, v=v), "v": lambda: paged.gather_paged(k_pages, v_pages, slots, k=k, v=v),
             "out": lambda: paged.paged_attention(q, k_pages, v_pages, table, lens, out=out)}
    names = {"k_pages": k_pages, "v_pages": v_pages, "q_out": out, "k": k, "v": v, "out": out}
    for name, call in calls.items():
        names[name].requires_grad_()
        with pytest.raises(RuntimeError, match=f"{name} requires a gradient"):
            call()
        names[name].requires_grad_(False)
    assert not launched
    k_pages.requires_grad_()
    with torch.no_grad():
        calls["k_pages"]()
    assert launched == ["cg_append_paged"]


def test_what_is_written_to_has_a_new_version(launched):
    """A backward pass that kept such a tensor refuses it then."""
    k, v, q, x = rows(6, 2, 64), rows(6, 2, 64), rows(6, 2, 64), rows(6, 2, 64)
    k_pages, v_pages, slots = rows(3, 4, 2, 64), rows(3, 4, 2, 64), on_gpu(torch.arange(6))
    tensors = (k, v, q, k_pages, v_pages)
    versions = [t._version for t in tensors]
    paged.append_paged(k, v, k_pages, v_pages, slots, q=q, q_out=q)
    assert [t._version - w for t, w in zip(tensors, versions)] == [0, 0, 1, 1, 1]
    paged.gather_paged(k_pages, v_pages, slots, k=k, v=v)
    assert [t._version - w for t, w in zip(tensors, versions)] == [1, 1, 1, 1, 1]
    weight = torch.ones((6, 2, 64), dtype=torch.float16, requires_grad=True)
    y = (weight * x).sum()
    paged.append_paged(k, v, k_pages, v_pages, slots, q=q, q_out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        pages = [rows(3, 4, 2, 64) for _ in range(2)]
        paged.append_paged(k, v, *pages, slots)
    paged.append_paged(k, v, *pages, slots)


def test_counts_beyond_32_bits_are_refused(launched, monkeypatch):
    """They would be cut off: 2^32 + 4 tokens would be 4."""
    T = 2 ** 32 + 4
    k, slots = rows(1, 2, 64), on_gpu(torch.zeros(1, dtype=torch.int64))
    k_pages, v_pages = (rows(3, 1, 2, 64).expand(3, T, 2, 64) for _ in range(2))  # pages of as many tokens, all the same memory
    lens, table = on_gpu(torch.ones(1, dtype=torch.int32)), on_gpu(torch.zeros((1, 1), dtype=torch.int32))
    monkeypatch.setattr(paged, "_turning", lambda *_: None)
    monkeypatch.setattr(paged, "_turns_for", lambda *_: (None, 0, 0, False, 0))
    x, at = (on_gpu(torch.empty(shape, dtype=dtype, device="meta")) for shape, dtype in (((T, 2, 64), torch.float16), ((T,), torch.int32)))
    for call in (lambda: paged.gather_paged(k_pages, v_pages, slots, k=k, v=rows(1, 2, 64)), lambda: paged.paged_attention(k, k_pages, v_pages, table, lens),
                 lambda: paged.apply_rotary(x, at, object())):
        with pytest.raises(RuntimeError, match="more than a call takes"):
            call()
    assert not launched


def test_jobs_of_nearly_two_to_the_31_tokens_or_layers_are_refused():
    """A block counts on to the end of its share of the tokens, behind the last."""
    from test_paged_refusals import rows_job
    L = _lib.lib()
    for entry in (L.cg_rotary, L.cg_append_paged, L.cg_gather_paged):
        for given in ({"ntokens": 2 ** 31 - 1}, {"ntokens": 2 ** 31 - 512}, {"nlayers": 2 ** 31 - 1}):
            assert entry(rows_job(**given), None) == -2, given


def test_views_that_negate_are_refused(launched):
    """The kernels read the memory as it is."""
    k, v, q = rows(6, 2, 64), rows(6, 2, 64), rows(6, 2, 64)
    pages, slots = (rows(3, 4, 2, 64), rows(3, 4, 2, 64)), on_gpu(torch.arange(6))
    table, lens = on_gpu(torch.zeros((6, 1), dtype=torch.int32)), on_gpu(torch.ones(6, dtype=torch.int32))
    neg = torch._neg_view
    for call in (lambda: paged.append_paged(neg(k), v, *pages, slots), lambda: paged.append_paged(k, v, *pages, neg(slots)),
                 lambda: paged.append_paged(k, v, *pages, slots, q=neg(q)), lambda: paged.gather_paged(neg(pages[0]), pages[1], slots, k=k, v=v),
                 lambda: paged.gather_paged(*pages, slots, k=neg(k), v=v), lambda: paged.paged_attention(neg(q), *pages, table, lens),
                 lambda: paged.paged_attention(q, *pages, neg(table), lens), lambda: paged.paged_attention(q, *pages, table, neg(lens))):
        with pytest.raises(RuntimeError, match="negates"):
            call()
    assert not launched
