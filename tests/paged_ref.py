"""The operators of a paged cache in 64 bits, on tensors of any device, and how far a kernel's rounding may take it from them."""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def turned(x, positions, frequencies, rot, interleaved, inverse=False):
    """x [..., T, H, D] in 64 bits, turned to positions [T] or [n, T]."""
    x = x.double().clone()
    if not rot:
        return x
    w = torch.tensor(frequencies, dtype=torch.float64, device=x.device)
    angle = (positions.double()[..., None] * w)[..., None, :] * (-1 if inverse else 1)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    xa, xb = x[..., a].clone(), x[..., b].clone()
    x[..., a] = xa * angle.cos() - xb * angle.sin()
    x[..., b] = xb * angle.cos() + xa * angle.sin()
    return x


def turned_tolerance(x, want, rot, interleaved, dtype):
    """One rounding of the result: half a step of it (of the smallest normal number, where it is smaller).  In front of it cosine and
    sine are each off by at most 2^-22 (a phase of 24 bits, half a turn long: pi 2^-25, and 4 units of the last place of a
    32-bit sine), products and the sum by 3 * 2^-24 of |x_a| + |x_b|: together below 2^-20 of that."""
    pair = x.double().abs().clone()
    if rot:
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        both = pair[..., a] + pair[..., b]
        pair[..., a], pair[..., b] = both, both
    tiny = torch.finfo(dtype).smallest_normal
    return half_step(dtype) * want.abs().clamp(min=tiny) * (1 + 2 ** -10) + 2.0 ** -20 * pair


def attention(q, k_pages, v_pages, table, lens, scale, causal=True, window=0):
    """(out, lse, tolerance) in 64 bits; lens: (first row, rows, keys) of every request; rows of no request are NaN.

    Tolerance of a value: half a step of the result, and of every weight (it is rounded to the cache's type in front of the second
    product), so 2 half steps of A = sum w |v| / sum w at most; a weight of fp16 below the normal numbers is off by up to 2^-25
    of the largest one; 32-bit sums of D products and of all keys: (D + 8) 2^-24 of scale sum |q_d k_d| in every score, which
    changes weights (and with them sum w) by that share, and (keys + 16) 2^-24 of A."""
    R, Q, D = q.shape
    page, H = k_pages.shape[1], k_pages.shape[2]
    group = Q // H
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    lse = torch.full((R, Q), math.nan, dtype=torch.float64, device=q.device)
    tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    h2 = half_step(q.dtype)
    for b, (first, n, kv) in enumerate(lens):
        j = torch.arange(kv, device=q.device)
        pages = table[b].to(q.device).long()[j // page]
        k, v = k_pages[pages, j % page].double(), v_pages[pages, j % page].double()  # [kv, H, D]
        for i in range(n):
            place = kv - n + i
            lo = max(0, place - window + 1) if window else 0
            hi = max(0, min(kv, place + 1)) if causal else kv
            if hi <= lo:
                out[first + i], lse[first + i] = 0.0, -math.inf
                continue
            x = q[first + i].double().view(H, group, D)
            s = torch.einsum("hgd,khd->hgk", x, k[lo:hi]) * scale
            size = (torch.einsum("hgd,khd->hgk", x.abs(), k[lo:hi].abs()) * abs(scale)).amax(-1)
            whole = torch.logsumexp(s, -1)
            w = torch.exp(s - whole[..., None])
            o = torch.einsum("hgk,khd->hgd", w, v[lo:hi])
            A = torch.einsum("hgk,khd->hgd", w, v[lo:hi].abs())
            score = ((D + 8) * 2.0 ** -24 * size)[..., None]
            t = h2 * o.abs() + A * (h2 * 1.02 + 2.02 * score + (hi - lo + 16) * 2.0 ** -24)
            if q.dtype == torch.float16:
                # weights relative to the largest: w / max w below 2^-14 is rounded to a multiple of 2^-24
                t += 2.0 ** -25 * w.amax(-1)[..., None] * v[lo:hi].abs().sum(0)[:, None, :]
                t += 2.0 ** -25  # the result, where it is below the normal numbers
            out[first + i], lse[first + i], tol[first + i] = o.reshape(Q, D), whole.reshape(Q), t.reshape(Q, D)
    return out, lse, tol
