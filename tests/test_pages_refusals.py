"""What the calls on pages and beams refuse, before anything is launched: through the C ABI without a GPU, and in Python."""
import ctypes
import os
import subprocess

import pytest
import torch

from cachegen_b200 import _lib, paged

P = 1 << 12  # an address that is never used: every call below is refused


def job_of(kind, pointers, **given):
    job = kind()
    for name in pointers.split():
        setattr(job, name, P)
    for name, value in given.items():
        setattr(job, name, value)
    return ctypes.byref(job)


def pages_job(**given):
    return job_of(_lib.PagesJob, "table kv_lens refs which new_table new_lens moves places q_starts slots workspace",
                  **{**dict(workspace_bytes=1 << 40, table_row=8, new_table_row=8, num_pages=100, nrows=4, width=8, page_size=16, nnew=6, ntokens=4), **given})


def copy_job(**given):
    return job_of(_lib.CopyJob, "pages_k pages_v src dst", **{**dict(num_pages=100, nlayers=2, ncopies=3, page_size=16, heads=2, head_size=64), **given})


def beam_job(**given):
    return job_of(_lib.BeamJob, "logits scores out_scores tokens parents workspace",
                  **{**dict(workspace_bytes=1 << 40, row_stride=100, dtype=0, nrequests=2, beams=3, vocab=100, k=4), **given})


def test_pages_jobs_are_refused():
    L = _lib.lib()
    calls = {"fork": lambda j: L.cg_fork_pages(j, None, None), "free": lambda j: L.cg_free_pages(j, None), "extend": lambda j: L.cg_extend_pages(j, None),
             "compact": lambda j: L.cg_compact_pages(j, None, None)}
    for name, call in calls.items():
        assert call(None) == -1
        for given, code in (({"nrows": -1}, -2), ({"width": -1}, -2), ({"page_size": 0}, -2), ({"num_pages": -1}, -2), ({"num_pages": 1 << 31}, -2), ({"nnew": -1}, -2),
                            ({"ntokens": -1}, -2), ({"nrows": 4097}, -6), ({"width": 1 << 28}, -2), ({"table": None}, -1), ({"kv_lens": None}, -1), ({"refs": None}, -1)):
            assert call(pages_job(**given)) == code, (name, given)
        if name != "free":
            for given, code in (({"workspace": None}, -6), ({"workspace_bytes": 1000}, -6), ({"workspace": P + 8}, -5)):
                assert call(pages_job(**given)) == code, (name, given)
    for given, code in (({"nnew": 4097}, -6), ({"which": None}, -1), ({"new_table": None}, -1), ({"new_lens": None}, -1), ({"moves": None}, -1)):
        assert calls["fork"](pages_job(**given)) == code, given
    assert calls["free"](pages_job(nnew=4097)) == -6 and calls["free"](pages_job(nnew=0)) == 0 and calls["free"](pages_job(which=None, nrows=0)) == 0
    assert calls["extend"](pages_job(slots=None)) == -1 and calls["extend"](pages_job(q_starts=None, ntokens=5)) == -2
    assert calls["extend"](pages_job(nrows=0)) == -2 and calls["extend"](pages_job(nrows=0, ntokens=0)) == 0
    assert calls["compact"](pages_job(places=None)) == -1 and calls["compact"](pages_job(moves=None)) == -1 and calls["compact"](pages_job(num_pages=0)) == 0
    for entry in (L.cg_fork_pages, L.cg_compact_pages):
        for given, code in (({"page_size": 8}, -2), ({"num_pages": 99}, -2), ({"pages_k": None}, -1), ({"pages_v": None}, -1), ({"heads": 0}, -2)):
            assert entry(pages_job(), copy_job(**given), None) == code, given
    assert L.cg_fork_pages(pages_job(nrows=0, nnew=0), None, None) == 0
    assert L.cg_pages_workspace(-1) == -2 and L.cg_pages_workspace(1 << 31) == -2 and L.cg_pages_workspace(0) > 0


def test_copies_are_refused():
    L = _lib.lib()
    assert L.cg_copy_pages(None, None) == -1
    for given, code in (({"ncopies": -1}, -2), ({"nlayers": -1}, -2), ({"page_size": 0}, -2), ({"heads": 0}, -2), ({"head_size": 0}, -2), ({"num_pages": -1}, -2),
                        ({"page_size": 1 << 20, "heads": 64}, -6), ({"pages_k": P + 1}, -5), ({"pages_v": P + 1}, -5), ({"nlayers": 1 << 30}, -6), ({"pages_k": None}, -1), ({"pages_v": None}, -1), ({"src": None}, -1), ({"dst": None}, -1)):
        assert L.cg_copy_pages(copy_job(**given), None) == code, given
    assert L.cg_copy_pages(copy_job(ncopies=0), None) == 0 and L.cg_copy_pages(copy_job(nlayers=0), None) == 0


def test_beam_jobs_are_refused():
    L = _lib.lib()
    assert L.cg_beam_select(None, None) == -1 and L.cg_beam_workspace(None) == -1
    for given, code in (({"dtype": 3}, -7), ({"dtype": -1}, -7), ({"nrequests": -1}, -2), ({"beams": 0}, -2), ({"vocab": 0}, -2), ({"vocab": (1 << 24) + 1}, -2), ({"k": 0}, -2),
                        ({"beams": 257}, -6), ({"k": 129}, -6), ({"beams": 100, "k": 100}, -6), ({"nrequests": 1 << 20}, -6)):
        assert L.cg_beam_select(beam_job(**given), None) == code, given
        assert L.cg_beam_workspace(beam_job(**given)) == code, given
    for given, code in (({"logits": None}, -1), ({"scores": None}, -1), ({"out_scores": None}, -1), ({"tokens": None}, -1), ({"parents": None}, -1), ({"workspace": None}, -6),
                        ({"workspace_bytes": 10}, -6), ({"workspace": P + 8}, -5), ({"logits": P + 1}, -5), ({"logits": P + 2, "dtype": 2}, -5)):
        assert L.cg_beam_select(beam_job(**given), None) == code, given
    assert L.cg_beam_select(beam_job(nrequests=0), None) == 0 and L.cg_beam_workspace(beam_job(nrequests=0)) == 0


def test_structures_have_the_sizes_of_the_header(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"cg_pages_job": (_lib.PagesJob, "nrows"), "cg_copy_job": (_lib.CopyJob, "wide"), "cg_beam_job": (_lib.BeamJob, "k")}
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cachegen_b200.h"\nint main(void) { ' + "".join(
        f'printf("%zu %zu\\n", sizeof({n}), offsetof({n}, {field}));' for n, (_, field) in names.items()) + " return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [x for kind, field in names.values() for x in (ctypes.sizeof(kind), getattr(kind, field).offset)]


def test_cpu_tensors_are_refused():
    k, i, f = torch.zeros((3, 4, 1, 8), dtype=torch.float16), torch.zeros(3, dtype=torch.int32), torch.zeros((1, 2))
    for call in (lambda: paged.copy_pages(k, k.clone(), i, i), lambda: paged.fork_pages(i[:, None], i, i, i, page_size=4), lambda: paged.free_pages(i[:, None], i, i, 4),
                 lambda: paged.extend_pages(i[:, None], i, i, 4), lambda: paged.compact_pages(i[:, None], i, i, page_size=4), lambda: paged.beam_select(f, f)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


GPU = pytest.mark.gpu


def tables():
    c = dict(device="cuda", dtype=torch.int32)
    return dict(page_table=torch.tensor([[0, 1], [2, -1]], **c), kv_lens=torch.tensor([5, 3], **c), refs=torch.tensor([1, 1, 1, 0, 0], **c))


def caches():
    return [torch.zeros((5, 4, 1, 8), dtype=torch.float16, device="cuda") for _ in range(2)]


TABLE_CHANGES = [
    dict(page_table=lambda t: t.long()), dict(page_table=lambda t: t[0]), dict(page_table=lambda t: t[:1]), dict(page_table=lambda t: t.cpu()),
    dict(page_table=lambda t: t.t().contiguous().t()), dict(kv_lens=lambda t: t.long()), dict(kv_lens=lambda t: t[:1]), dict(kv_lens=lambda t: t.cpu()),
    dict(refs=lambda t: t.long()), dict(refs=lambda t: t[::2]), dict(refs=lambda t: t[None])]


@GPU
@pytest.mark.parametrize("change", TABLE_CHANGES)
def test_tables_are_refused(change):
    given = tables()
    for name, how in change.items():
        given[name] = how(given[name])
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (lambda: paged.fork_pages(given["page_table"], given["kv_lens"], i, given["refs"], page_size=4), lambda: paged.free_pages(**given, page_size=4),
                 lambda: paged.extend_pages(**given, page_size=4), lambda: paged.compact_pages(**given, page_size=4)):
        with pytest.raises(RuntimeError):
            call()


@GPU
def test_what_does_not_go_together_is_refused():
    t, (k, v), i = tables(), caches(), torch.zeros(2, dtype=torch.int32, device="cuda")
    args = t["page_table"], t["kv_lens"], i, t["refs"]
    rows = t["page_table"], t["kv_lens"], t["refs"]
    kept = {n: x.clone() for n, x in t.items()}
    for call in (
            lambda: paged.fork_pages(*args), lambda: paged.fork_pages(*args, k), lambda: paged.fork_pages(*args, k, v, page_size=8), lambda: paged.fork_pages(*args, k[:4], v[:4]),
            lambda: paged.fork_pages(*args, k, v[:, :2]), lambda: paged.fork_pages(*args, k, k), lambda: paged.fork_pages(*args, k, v.bfloat16()),
            lambda: paged.fork_pages(t["page_table"], t["kv_lens"], i.float(), t["refs"], k, v), lambda: paged.fork_pages(t["page_table"], t["kv_lens"], i[None], t["refs"], k, v),
            lambda: paged.fork_pages(*args, k, v, out=(t["page_table"], t["kv_lens"].clone())), lambda: paged.fork_pages(*args, k, v, out=(t["page_table"].clone(), t["kv_lens"])),
            lambda: paged.fork_pages(*args, k, v, out=(t["page_table"].clone()[:1], t["kv_lens"].clone())), lambda: paged.fork_pages(*args, page_size=0),
            lambda: paged.fork_pages(t["page_table"], t["kv_lens"], torch.zeros(4097, dtype=torch.int32, device="cuda"), t["refs"], page_size=4),
            lambda: paged.fork_pages(*args, page_size=2 ** 30), lambda: paged.fork_pages(*args, k.requires_grad_(), v), lambda: paged.free_pages(*rows, 0), lambda: paged.free_pages(*rows, 4, rows=i.float()),
            lambda: paged.free_pages(*rows, 4, rows=t["kv_lens"]), lambda: paged.extend_pages(*rows, 4, tokens=3), lambda: paged.extend_pages(*rows, 4, q_starts=torch.zeros(3, dtype=torch.int32, device="cuda")),
            lambda: paged.extend_pages(*rows, 4, q_starts=i, tokens=3), lambda: paged.extend_pages(*rows, 4, q_starts=torch.zeros(3, device="cuda"), tokens=3),
            lambda: paged.extend_pages(t["page_table"], t["kv_lens"], t["refs"][:0].expand(0), 0), lambda: paged.extend_pages(t["refs"][:2].view(2, 1), t["kv_lens"], t["refs"], 4),
            lambda: paged.compact_pages(*rows), lambda: paged.compact_pages(*rows, v[:3], v[2:]), lambda: paged.copy_pages(v, v, i, i), lambda: paged.copy_pages(v, caches()[0], i, i.long()),
            lambda: paged.copy_pages(v, caches()[0], i, i[:1]), lambda: paged.copy_pages(v, caches()[0], i, i, tokens=i.long()), lambda: paged.copy_pages(v, caches()[0], i[None], i[None]),
            lambda: paged.copy_pages(v.float(), v.float(), i, i), lambda: paged.copy_pages(v[:1].expand(5, 4, 1, 8), caches()[0], i, i)):
        with pytest.raises(RuntimeError):
            call()
    assert all(torch.equal(x, kept[n]) for n, x in t.items())


@GPU
def test_beams_are_refused():
    x, s = torch.zeros((6, 40), dtype=torch.float16, device="cuda"), torch.zeros((2, 3), device="cuda")
    paged.beam_select(x, s, 4)
    for call in (lambda: paged.beam_select(x.double(), s, 4), lambda: paged.beam_select(x, s.double(), 4), lambda: paged.beam_select(x, s.cpu(), 4), lambda: paged.beam_select(x[:5], s, 4),
                 lambda: paged.beam_select(x, s[0], 4), lambda: paged.beam_select(x, s, 0), lambda: paged.beam_select(x, s, 129), lambda: paged.beam_select(x, s, -1),
                 lambda: paged.beam_select(x[:, :0], s, 4), lambda: paged.beam_select(x.view(2, 3, 40), s, 4), lambda: paged.beam_select(x.t().contiguous().t(), s, 4),
                 lambda: paged.beam_select(x.float().requires_grad_(), s, 4), lambda: paged.beam_select(x, s.clone().requires_grad_(), 4), lambda: paged.beam_select(x, torch.zeros((3, 2), device="cuda").t(), 4),
                 lambda: paged.beam_select(x.expand(6, 40)[:0], torch.zeros((0, 0), device="cuda"), 4)):
        with pytest.raises(RuntimeError):
            call()
