"""The 8-bit key/value cache in 64 bits, from its definition, a sequence and a
head at a time (torch on the CPU)."""
from __future__ import annotations

import math

import torch


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """The e4m3 number nearest to x, ties to even: 4 significant bits, the
    smallest step 2^-9 (|x| <= 448; NaN stays NaN)."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def codes(values: torch.Tensor) -> torch.Tensor:
    """e4m3 numbers as their bytes."""
    return values.float().to(torch.float8_e4m3fn).view(torch.uint8)


def values(codes: torch.Tensor) -> torch.Tensor:
    return codes.view(torch.float8_e4m3fn).double()


def scale_of(amax: float) -> float:
    """The smallest power of two s >= 2^-110 with amax <= 448 s."""
    s = 2.0 ** -110
    while amax > 448 * s:
        s *= 2
    return s


def tokens(code, scale, pages, n):
    """The first n tokens in these pages of one head: [n, d]."""
    if n == 0:
        return torch.zeros(0, code.shape[-1], dtype=torch.float64)
    return torch.cat([values(code[p]) * float(scale[p]) for p in pages])[:n]


def append(cache, k, v, table, lengths, starts):
    """cache: CPU (k, v, k_scale, v_scale), written in place."""
    page = cache[0].shape[2]
    for b, total in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        for head in range(cache[0].shape[1]):
            for code, scale, x, other in ((cache[0], cache[2], k, v), (cache[1], cache[3], v, None)):
                for i in range((total - n) // page, -(-total // page) if n else 0):
                    p = table[b][i]
                    lo, hi = max(0, total - n - i * page), min(page, total - i * page)
                    first = starts[b] + i * page + lo - (total - n)
                    new = x[first: first + hi - lo, head].double()
                    fine = torch.isfinite(new)
                    s = scale_of(float(torch.where(fine, new.abs(), 0.0).max()))
                    if lo:
                        s = max(s, float(scale[p, head]))
                        old = values(code[p, head, :lo]) * (float(scale[p, head]) / s)
                        code[p, head, :lo] = codes(e4m3(old))
                    got = e4m3(torch.where(fine, new, 0.0) / s)
                    if other is not None:  # a key of a token with a bad element
                        bad = ~(fine & torch.isfinite(other[first: first + hi - lo, head])).all(1)
                        got[bad] = math.nan
                    code[p, head, lo:hi] = codes(got)
                    scale[p, head] = s


def attention(q, cache, table, lengths, starts, scale, weights=None, lse=None):
    """(out, lse, size): size bounds what rounding can do to out: per output the
    weights' sum of |v|, and per row the largest sum of |q k| scale.  With
    `weights` (and lse) they are added to instead, in place."""
    page, heads = cache[0].shape[2], cache[0].shape[1]
    T, H, D = q.shape
    out = torch.zeros(T, H, D, dtype=torch.float64)
    log = torch.full((T, H), -math.inf, dtype=torch.float64)
    mass, reach = torch.zeros_like(out), torch.zeros(T, H, dtype=torch.float64)
    for b, total in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        pages = table[b][: -(-total // page)]
        at = torch.arange(total - n, total)
        see = torch.arange(total)[None] <= at[:, None]
        for h in range(H):
            g = h // (H // heads)
            kk = tokens(cache[0][:, g], cache[2][:, g], pages, total)
            vv = tokens(cache[1][:, g], cache[3][:, g], pages, total)
            x = q[starts[b]: starts[b + 1], h].double()
            s = torch.where(see, (x @ kk.t()) * scale, -math.inf)
            span = slice(starts[b], starts[b + 1])
            if total:
                reach[span, h] = torch.where(see, (x.abs() @ kk.abs().t()) * abs(scale), 0.0).amax(1)
            if weights is not None:
                p = torch.where(see, torch.exp(s - lse[span, h, None].double()), 0.0)
                weights[b, g, :total] += p.sum(0)
                continue
            log[span, h] = torch.logsumexp(s, 1) if total else log[span, h]
            p = torch.where(see, torch.exp(s - log[span, h, None]), 0.0)
            out[span, h] = p @ vv
            mass[span, h] = p @ vv.abs()
    return out, log, (mass, reach)


def evict(cache, weights, table, new_table, lengths, keep, recent, sink):
    """Writes the new pages of the CPU cache; (kept, new lengths, new weights)."""
    page, heads = cache[0].shape[2], cache[0].shape[1]
    kept = torch.full((len(lengths), heads, keep), -1, dtype=torch.int32)
    moved = torch.zeros_like(weights)
    for b, total in enumerate(lengths):
        left = min(total, keep)
        for h in range(heads):
            rank = []
            for i in range(total):
                w = float(weights[b, h, i])
                w = -math.inf if math.isnan(w) else w
                forced = i < sink or i >= total - recent
                rank.append((0 if forced else 1, -w, i))
            at = sorted(i for _, _, i in sorted(rank)[:left]) if total > keep else list(range(total))
            kept[b, h, :left] = torch.tensor(at, dtype=torch.int32)
            moved[b, h, :left] = weights[b, h, at]
            for code, scale in ((cache[0], cache[2]), (cache[1], cache[3])):
                x = tokens(code[:, h], scale[:, h], table[b][: -(-total // page)], total)[at]
                for i in range(-(-left // page)):
                    part, p = x[i * page: (i + 1) * page], new_table[b][i]
                    s = scale_of(float(torch.nan_to_num(part, nan=0.0).abs().max()))
                    code[p, h, : part.shape[0]] = codes(e4m3(part / s))
                    scale[p, h] = s
    return kept, [min(n, keep) for n in lengths], moved
