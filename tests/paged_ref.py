"""Plain 64-bit forms of the paged cache's operators, on CPU tensors, with bounds on how far a kernel
that holds its sums in 32 bits may be off."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def pages_of(n, page):
    return -(-n // page)


def plan(lens, add, table, free, num_free, page, tokens):
    """(slots, positions, starts, lens, num_free, table, free[:num_free]) after a step; the arguments stay."""
    table, free, lens = [list(r) for r in table], list(free), list(lens)
    before, top, slots, positions, starts = list(lens), num_free, [], [], [0]
    for z, a in enumerate(add):
        if a < 0:
            for j in range(pages_of(lens[z], page)):
                free[top] = table[z][j]
                top += 1
            lens[z] = 0
    for z, a in enumerate(add):
        for _ in range(max(a, 0)):
            if lens[z] % page == 0:
                top -= 1
                assert top >= 0, "the step does not fit"
                table[z][lens[z] // page] = free[top]
            slots.append(table[z][lens[z] // page] * page + lens[z] % page)
            positions.append(lens[z])
            lens[z] += 1
        starts.append(len(slots))
    pad = tokens - len(slots)
    assert pad >= 0 and len(before) == len(lens)
    return slots + [-1] * pad, positions + [0] * pad, starts, lens, top, table, free[:top]


def keep(x, scale):
    """What an 8-bit cache keeps of ``x`` [tokens, heads, dim]: the 32-bit quotient, limited, rounded once."""
    return (x.float() / scale.float().view(1, -1, 1)).clamp(-448.0, 448.0).to(E4M3)


def attention(q, k_cache, v_cache, table, lens, sm_scale, starts=None, causal=True, window=0, k_scale=None, v_scale=None):
    """(out, lse, out_tolerance, lse_tolerance) in 64 bits; rows outside all requests are NaN in ``out``."""
    T, Hq, D = q.shape
    page, H = k_cache.shape[1:3]
    group = Hq // H
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    tol = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), math.nan, dtype=torch.float64)
    lse_tol = torch.zeros(T, Hq, dtype=torch.float64)
    half_step = torch.finfo(q.dtype).eps / 2
    for z in range(len(lens)):
        first, last = (z, z + 1) if starts is None else (starts[z], starts[z + 1])
        n, length = last - first, lens[z]
        ids = torch.tensor(table[z][: pages_of(length, page)], dtype=torch.long)
        if k_cache.dtype == E4M3:
            k, v = (c.view(torch.uint8)[ids].view(E4M3).double().reshape(-1, H, D)[:length] for c in (k_cache, v_cache))
            k, v = k * k_scale.double().view(1, -1, 1), v * v_scale.double().view(1, -1, 1)
        else:
            k, v = (c[ids].double().reshape(-1, H, D)[:length] for c in (k_cache, v_cache))
        for i in range(n):
            pos = length - n + i
            hi = min(length, pos + 1) if causal else length
            lo = max(0, pos - window + 1) if window else 0
            row = first + i
            if hi <= lo:
                out[row], lse[row] = 0.0, -math.inf
                continue
            qr = q[row].double().view(H, group, D)
            kk, vv = k[lo:hi], v[lo:hi]
            x = torch.einsum("hgd,lhd->hgl", qr, kk) * sm_scale
            p = torch.softmax(x, -1)
            out[row] = torch.einsum("hgl,lhd->hgd", p, vv).reshape(Hq, D)
            lse[row] = (torch.logsumexp(x, -1) / math.log(2.0)).reshape(Hq)
            # Score: D products summed in 32 bits, scaled and turned to base 2 (3 roundings), and the
            # subtraction of the maximum (one, of a value up to |x| / ln 2): an error of e in its exponent.
            # A weight is then off by a factor 1 + e + 2^-21 (exp2 and its argument's rounding), numerator
            # and sum alike; sums of m terms add m / 2^24 each; weights enter the product with at least 16
            # bits (2^-16).  All of that is relative to sum p |v|.
            m = hi - lo
            e = torch.einsum("hgd,lhd->hgl", qr.abs(), kk.abs()).amax(-1) * abs(sm_scale) * (D + 8) * 2.0 ** -24
            rel = 2 * e + 2.0 ** -20 + 2.0 ** -16 + (m + 64) * 2.0 ** -23
            size = torch.einsum("hgl,lhd->hgd", p, vv.abs())
            o_tol = size * rel[..., None]
            o_tol = o_tol + half_step * (out[row].view(H, group, D).abs() + o_tol)
            # Half a step among the smallest numbers of the type.
            tol[row] = o_tol.reshape(Hq, D) + torch.finfo(q.dtype).smallest_normal * half_step * 2
            lse_tol[row] = (e.reshape(Hq) + (m + 64) * 2.0 ** -24) * 1.5 + 2.0 ** -20 + lse[row].abs() * 2.0 ** -22
    return out, lse, tol, lse_tol
