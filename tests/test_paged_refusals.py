"""What the calls on a paged cache refuse, before anything is launched: through the C ABI without a GPU, and in Python on tensors
that only say that they are on one."""
import ctypes
import math
import subprocess

import pytest
import torch

from cachegen_b200 import _lib, paged

P = 1 << 12  # an address that is never used: every call below is refused


def rows_job(**given):
    job = _lib.RowsJob()
    for name in ("q", "q_out", "k", "v", "k_out", "pages_k", "pages_v", "positions", "slots", "turns"):
        setattr(job, name, P)
    job.dtype, job.nlayers, job.ntokens, job.heads, job.head_size, job.page_size, job.num_pages = 0, 1, 4, 2, 64, 16, 8
    for name, value in given.items():
        setattr(job, name, value)
    return ctypes.byref(job)


def test_rows_jobs_are_refused():
    L = _lib.lib()
    for entry in (L.cg_rotary, L.cg_append_paged, L.cg_gather_paged):
        assert entry(None, None) == -1
        for given, code in (({"dtype": 2}, -7), ({"head_size": 0}, -2), ({"head_size": 513}, -2), ({"nlayers": -1}, -2), ({"ntokens": -1}, -2),
                            ({"heads": -1}, -2), ({"rotary_dims": 3}, -2), ({"rotary_dims": 66}, -2), ({"rotary_dims": -2}, -2),
                            ({"rotary_dims": 64, "positions": None}, -1), ({"rotary_dims": 64, "turns": None}, -1), ({"heads": 32768, "q_heads": 1}, -2),
                            ({"k": None}, -1)):
            assert entry(rows_job(**given), None) == code, given
        assert entry(rows_job(ntokens=0), None) == 0 and entry(rows_job(nlayers=0), None) == 0  # nothing to do
    assert L.cg_rotary(rows_job(k_out=None), None) == -1
    for entry in (L.cg_append_paged, L.cg_gather_paged):
        for given, code in (({"v": None}, -1), ({"pages_k": None}, -1), ({"pages_v": None}, -1), ({"slots": None}, -1), ({"heads": 0}, -2),
                            ({"page_size": 0}, -2), ({"num_pages": -1}, -2), ({"pos_layer": 4}, -2)):
            assert entry(rows_job(**given), None) == code, given
    assert L.cg_append_paged(rows_job(q_heads=2, q=None), None) == -1
    assert L.cg_append_paged(rows_job(q_heads=2, nlayers=2), None) == -2


def attention_job(**given):
    job = _lib.AttentionJob()
    for name in ("q", "pages_k", "pages_v", "out", "table", "kv_lens", "q_starts", "workspace"):
        setattr(job, name, P)
    job.dtype, job.nrequests, job.nrows, job.q_heads, job.heads, job.head_size, job.page_size, job.table_width = 0, 2, 5, 8, 2, 64, 16, 40
    job.num_pages, job.table_row, job.workspace_bytes, job.scale = 100, 40, 1 << 40, 0.125
    for name, value in given.items():
        if isinstance(value, tuple):
            getattr(job, name)[:] = value
        else:
            setattr(job, name, value)
    return ctypes.byref(job)


def test_attention_jobs_are_refused():
    L = _lib.lib()
    assert L.cg_paged_attention(None, None) == -1 and L.cg_paged_attention_workspace(None) == -1
    for given, code in (({"dtype": 2}, -7), ({"nrequests": -1}, -2), ({"nrows": -1}, -2), ({"heads": 0}, -2), ({"q_heads": 0}, -2), ({"q_heads": 7}, -2),
                        ({"head_size": 0}, -2), ({"head_size": 136}, -2), ({"head_size": 68}, -5), ({"page_size": 0}, -2), ({"table_width": -1}, -2),
                        ({"num_pages": -1}, -2), ({"num_pages": 1 << 31}, -2), ({"window": -1}, -2), ({"max_q": -1}, -2), ({"nrows": 1 << 29}, -2),
                        ({"q_starts": None}, -2), ({"nrequests": 4097}, -6), ({"nrows": 1 << 27, "table_width": 1 << 21}, -6)):
        assert L.cg_paged_attention(attention_job(**given), None) == code, given
        assert L.cg_paged_attention_workspace(attention_job(**given)) == code, given
    for given, code in (({"q": None}, -1), ({"out": None}, -1), ({"kv_lens": None}, -1), ({"table": None}, -1), ({"pages_k": None}, -1), ({"pages_v": None}, -1),
                        ({"q": P + 8}, -5), ({"out": P + 2}, -5), ({"pages_k": P + 8}, -5), ({"workspace": P + 8}, -5), ({"q_strides": (4, 8)}, -5),
                        ({"out_strides": (8, 12)}, -5), ({"pages_k_strides": (8, 8, 2)}, -5), ({"pages_v_strides": (1, 8, 8)}, -5),
                        ({"workspace": None}, -6), ({"workspace_bytes": 100}, -6)):
        assert L.cg_paged_attention(attention_job(**given), None) == code, given
    assert L.cg_paged_attention(attention_job(nrows=0, nrequests=0), None) == 0 and L.cg_paged_attention_workspace(attention_job(nrows=0)) == 0


def test_structures_have_the_sizes_of_the_header(tmp_path):
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cachegen_b200.h"\nint main(void) { printf("%zu %zu %zu %zu\\n", sizeof(cg_rows_job), '
                   'offsetof(cg_rows_job, dtype), sizeof(cg_attention_job), offsetof(cg_attention_job, scale)); return 0; }\n')
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.RowsJob), _lib.RowsJob.dtype.offset, ctypes.sizeof(_lib.AttentionJob), _lib.AttentionJob.scale.offset]


def test_frequencies():
    r = paged.Rotary(128)
    assert r.frequencies[0] == 1.0 and math.isclose(r.frequencies[-1], 10000.0 ** (-126 / 128)) and len(r.frequencies) == 64
    assert paged.Rotary(128, rotary_dims=32).frequencies == paged.Rotary(32).frequencies
    linear = paged.Rotary(64, scaling=("linear", 4.0)).frequencies
    assert all(math.isclose(a * 4.0, b) for a, b in zip(linear, paged.Rotary(64).frequencies))
    ntk = paged.Rotary(64, scaling=("ntk", 4.0)).frequencies
    assert ntk[0] == 1.0 and math.isclose(ntk[-1] * 4.0, paged.Rotary(64).frequencies[-1])
    bands = paged.Rotary(64, scaling=("bands", 8.0, 1.0, 4.0, 8192)).frequencies
    plain = paged.Rotary(64).frequencies
    assert bands[0] == plain[0] and math.isclose(bands[-1] * 8.0, plain[-1]) and all(b <= a for a, b in zip(plain, bands))
    # the turns that a kernel multiplies with: 2^-64 of a turn and the rounding of the frequency itself
    for w, t in zip(r.frequencies, r._turns.tolist()):
        assert abs(t % 2 ** 64 / 2 ** 64 - w / (2 * math.pi)) < 2 ** -52


@pytest.mark.parametrize("given", [
    dict(head_size=0), dict(head_size=63), dict(head_size=64, rotary_dims=65), dict(head_size=64, rotary_dims=66), dict(head_size=64, rotary_dims=0),
    dict(head_size=64, base=0.0), dict(head_size=64, scaling=("cubic", 2.0)), dict(head_size=64, scaling=("linear",)), dict(head_size=64, scaling=("linear", 0.0)),
    dict(head_size=64, scaling=("linear", 2.0, 3.0)), dict(head_size=64, scaling=("bands", 8.0, 4.0, 1.0, 8192)), dict(head_size=2, scaling=("ntk", 2.0)),
    dict(head_size=8, frequencies=[1.0]), dict(head_size=4, frequencies=[1.0, math.inf]), dict(head_size=4, frequencies=[1.0, 2.0], scaling=("linear", 2.0))])
def test_rotary_settings_are_refused(given):
    with pytest.raises(ValueError):
        paged.Rotary(**given)


def test_cpu_tensors_are_refused():
    t = torch.zeros((2, 2, 64), dtype=torch.float16)
    pages = torch.zeros((2, 4, 2, 64), dtype=torch.float16)
    at = torch.zeros(2, dtype=torch.int64)
    r = paged.Rotary(64)
    for call in (lambda: paged.apply_rotary(t, at, r), lambda: paged.append_paged(t, t, pages, pages, at),
                 lambda: paged.gather_paged(pages, pages, at), lambda: paged.paged_attention(t, pages, pages, at.int()[:, None], at.int())):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


GPU = pytest.mark.gpu


def tensors():
    c = dict(device="cuda", dtype=torch.float16)
    return dict(k=torch.zeros((3, 2, 64), **c), v=torch.zeros((3, 2, 64), **c), k_pages=torch.zeros((4, 16, 2, 64), **c),
                v_pages=torch.zeros((4, 16, 2, 64), **c), slots=torch.arange(3, device="cuda"))


@GPU
@pytest.mark.parametrize("change", [
    dict(k=lambda t: t.float()), dict(v=lambda t: t.bfloat16()), dict(k=lambda t: t[0]), dict(v=lambda t: t[:2]), dict(k_pages=lambda t: t.bfloat16()),
    dict(k_pages=lambda t: t[:, :, :1]), dict(v_pages=lambda t: t[..., :32]), dict(v_pages=lambda t: t[:3]), dict(k_pages=lambda t: t[0]),
    dict(slots=lambda t: t[:2]), dict(slots=lambda t: t.float()), dict(slots=lambda t: t.cpu()), dict(v_pages=lambda t: t.cpu()),
    dict(k_pages=lambda t: t[:1].expand(4, 16, 2, 64)), dict(k=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)),
    dict(k=lambda t: t.requires_grad_())])
def test_append_refuses(change):
    given = tensors()
    for name, how in change.items():
        given[name] = how(given[name])
    with pytest.raises(RuntimeError):
        paged.append_paged(**given)


@GPU
def test_append_refuses_what_does_not_go_together():
    r, t = paged.Rotary(64), tensors()
    at = torch.arange(3, device="cuda")
    for more in (dict(rotary=r), dict(positions=at), dict(rotary=paged.Rotary(128), positions=at), dict(rotary=r, positions=at[:2]), dict(q_out=t["k"]),
                 dict(q=t["k"][:2]), dict(q=t["k"], q_out=t["k"][:, :, :32]), dict(rotary=r, positions=at.float())):
        with pytest.raises(RuntimeError):
            paged.append_paged(**t, **more)
    with pytest.raises(RuntimeError, match="same memory"):
        paged.append_paged(t["k"], t["v"], t["k_pages"], t["k_pages"], t["slots"])
    buffer = torch.zeros((4, 2, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        paged.append_paged(**t, q=buffer[:3], q_out=buffer[1:])
    with pytest.raises(RuntimeError, match="overlap"):
        paged.append_paged(t["k_pages"][0, :3], t["v"], t["k_pages"], t["v_pages"], t["slots"])
    with pytest.raises(RuntimeError, match="overlap"):
        paged.gather_paged(t["k_pages"], t["v_pages"], t["slots"], k=t["k_pages"][0, :3])
    with pytest.raises(RuntimeError):
        paged.gather_paged(t["k_pages"], t["v_pages"], t["slots"], k=t["k"][:2])
    layers = {n: x[None] for n, x in t.items() if n != "slots"}
    with pytest.raises(RuntimeError, match="one layer"):
        paged.append_paged(**layers, slots=t["slots"], q=t["k"])


@GPU
def test_rotary_refuses():
    x = torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda")
    at, r = torch.arange(3, device="cuda"), paged.Rotary(64)
    for call in (lambda: paged.apply_rotary(x, at, None), lambda: paged.apply_rotary(x, at[:2], r), lambda: paged.apply_rotary(x[0], at, r),
                 lambda: paged.apply_rotary(x, at, paged.Rotary(32)), lambda: paged.apply_rotary(x, at, r, out=x[:2]),
                 lambda: paged.apply_rotary(x.float(), at, r), lambda: paged.apply_rotary(x, at.cpu(), r)):
        with pytest.raises(RuntimeError):
            call()


@GPU
@pytest.mark.parametrize("change", [
    dict(q=lambda t: t.float()), dict(q=lambda t: t.bfloat16()), dict(q=lambda t: t[0]), dict(q=lambda t: t[:, :3]), dict(q=lambda t: t[..., :32]),
    dict(q=lambda t: torch.zeros((3, 4, 66), dtype=torch.float16, device="cuda")[..., 1:65]), dict(k_pages=lambda t: t[..., :32]),
    dict(v_pages=lambda t: t[:2]), dict(page_table=lambda t: t.long()), dict(page_table=lambda t: t[:1]), dict(kv_lens=lambda t: t.long()),
    dict(kv_lens=lambda t: t[:1]), dict(q_starts=lambda t: t[:2]), dict(q_starts=lambda t: None), dict(q_starts=lambda t: t.cpu()),
    dict(page_table=lambda t: t.cpu()), dict(window=lambda t: -1), dict(max_q=lambda t: -1), dict(out=lambda t: torch.zeros_like(t)[:1]),
    dict(q=lambda t: t.requires_grad_())])
def test_attention_refuses(change):
    c = dict(device="cuda", dtype=torch.int32)
    given = dict(q=torch.zeros((3, 4, 64), dtype=torch.float16, device="cuda"), k_pages=tensors()["k_pages"], v_pages=tensors()["v_pages"],
                 page_table=torch.zeros((2, 2), **c), kv_lens=torch.full((2,), 5, **c), q_starts=torch.tensor([0, 1, 3], **c), window=0, max_q=0)
    given["out"] = torch.zeros_like(given["q"])
    paged.paged_attention(**given)
    for name, how in change.items():
        given[name] = how(given[name])
    with pytest.raises(RuntimeError):
        paged.paged_attention(**given)


def test_turns_are_rounded_to_nearest():
    import random
    from fractions import Fraction
    rng = random.Random(1)
    for w in [1.0, 0.5, 1e-7, 1e-300, -0.25, 7.0, 0.0] + [rng.uniform(-1, 1) * 10.0 ** rng.randint(-12, 3) for _ in range(300)]:
        assert paged._turns(w) == round(Fraction(w) / paged._TWO_PI * 2 ** 64) % 2 ** 64
