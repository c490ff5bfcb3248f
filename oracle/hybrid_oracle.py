"""Plain 64-bit definitions, on the CPU, of what surrounds the recurrent step in a hybrid model's layer: the 8-bit
key/value cache (append, attention) and the layer norm with 8-bit output.  Test infrastructure, written from the formulas."""

from __future__ import annotations

import math

import torch

F8 = torch.float8_e4m3fn
F8_MAX = 448.0


def power_of_two_scale(amax: float) -> float:
    """The smallest power of two s with amax / s <= 448, within 2^-100 .. 2^119."""
    if amax == 0.0:
        return 2.0 ** -100
    part, power = math.frexp(amax / F8_MAX)             # part in [0.5, 1)
    power -= part == 0.5
    return 2.0 ** min(max(power, -100), 119)


def rows_of(b, N, B, query_start):
    """First row and number of rows of request b."""
    if query_start is None:
        return b * (N // B), N // B
    first = min(max(int(query_start[b]), 0), N)
    return first, max(min(int(query_start[b + 1]), N) - first, 0)


def page_of(table, b, j, page, num_pages):
    p = int(table[b][j // page])
    return p if 0 < p < num_pages else 0


def append(k, v, cache, table, lengths, query_start=None):
    """Returns the cache as it is after the append; ``cache`` itself is left alone."""
    kc, ks, vc, vs = (t.clone() for t in cache)
    pages, HKV, page, D = kc.shape
    block = page // ks.shape[2]
    N, B = k.shape[0], len(lengths)
    for b in range(B):
        first, n = rows_of(b, N, B, query_start)
        length = min(max(int(lengths[b]), 0), table.shape[1] * page)
        start = 0
        while start < n:
            pos = length - n + start
            if pos < 0:
                start += 1
                continue
            p, m = page_of(table, b, pos, page, pages), min(n - start, block - pos % block)
            if p:
                for h in range(HKV):
                    rows = slice(first + start, first + start + m)
                    xk, xv = k[rows, h].double(), v[rows, h].double()
                    fine = torch.isfinite(xk).all(1) & torch.isfinite(xv).all(1)
                    for x, codes, scale in ((xk, kc, ks), (xv, vc, vs)):
                        off, j = pos % page, pos % page // block
                        early = codes[p, h, off - pos % block:off]
                        s = power_of_two_scale(float(x[fine].abs().max()) if fine.any() else 0.0)
                        if pos % block:
                            old = float(scale[p, h, j])
                            if s > old:
                                early.copy_((early.float() * (old / s)).to(F8))
                            s = max(s, old)
                        scale[p, h, j] = s
                        y = (x / s).clamp(-F8_MAX, F8_MAX).float()
                        y[~fine] = math.nan if codes is kc else 0.0
                        codes[p, h, off:off + m] = y.to(F8)
            start += m
    return kc, ks, vc, vs


def attention(q, scale, cache, table, lengths, query_start=None):
    """(out, weight, size): the attention in 64 bits; the same with |v| in v's place; and the largest sum of magnitudes
    behind one of the row's scores -- what an error bound is made of."""
    kc, ks, vc, vs = cache
    pages, HKV, page, D = kc.shape
    block = page // ks.shape[2]
    N, HQ, _ = q.shape
    B = len(lengths)
    out, weight = torch.zeros(N, HQ, D, dtype=torch.float64), torch.zeros(N, HQ, D, dtype=torch.float64)
    size = torch.zeros(N, HQ, 1, dtype=torch.float64)
    kf, vf = ((c.float().double().view(pages, HKV, -1, block, D) * s.double()[..., None, None]).view(pages, HKV, page, D)
              for c, s in ((kc, ks), (vc, vs)))
    for b in range(B):
        first, n = rows_of(b, N, B, query_start)
        length = min(max(int(lengths[b]), 0), table.shape[1] * page)
        ids = torch.tensor([page_of(table, b, j, page, pages) for j in range(length)], dtype=torch.long)
        offs = torch.arange(length) % page
        for i in range(n):
            there = (ids > 0) & (torch.arange(length) <= length - n + i)
            if not there.any():
                continue
            at, off = ids[there], offs[there]
            for h in range(HQ):
                g = h // (HQ // HKV)
                x = q[first + i, h].double()
                K, V = kf[at, g, off], vf[at, g, off]
                p = torch.softmax(K @ x * scale, 0)
                out[first + i, h] = p @ V
                weight[first + i, h] = p @ V.abs()
                size[first + i, h] = abs(scale) * (K.abs() @ x.abs()).max()
    return out, weight, size


def add_rms_norm(x, residual, weight, eps, group):
    """(h, y, scale): the sum, the normed rows and their scales, in 64 bits."""
    h = x.double() + (0 if residual is None else residual.double())
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double()
    parts = y.split(group or y.shape[1], dim=1)
    scale = torch.stack([p.abs().amax(1).clamp(min=1e-12) / F8_MAX for p in parts], 1)
    return h, y, scale
