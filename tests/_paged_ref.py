"""Plain 64-bit statement of the paged cache's operators, row by row on the CPU, and
the inputs their tests share."""
from __future__ import annotations

import math

import torch

from _synth import randn


def tables(n, d):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * (
        1.0 / 500000.0 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))[None, :]
    return ang.cos().float(), ang.sin().float()


def rope32(x, cos, sin):
    """x [heads, d] in fp32 at one position's angles [d / 2], products rounded separately."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def pages_for(lens, S, seed, spare=3, width=None):
    """(pages, table): every row's pages in random order; -7 past a row's own."""
    need = [max(1, -(-max(n, 0) // S)) for n in lens]
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(sum(need) + spare, generator=g)
    table = torch.full((len(lens), width or max(need)), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n].int()
        at += n
    return len(ids), table


def gather(pages, row, h, n, S):
    """Tokens 0..n-1 of a head through a table row."""
    j = torch.arange(n)
    return pages[row.long()[j // S], h, j % S]


def attention(q, k, v, cos, sin, k_pages, v_pages, table, lengths, positions, weight):
    """(out, tolerance scale p @ |v|, score scale) in 64 bits and the
    weights afterwards; k_pages and v_pages are updated in place."""
    kp, vp = k_pages, v_pages
    P, nkv, S, d = kp.shape
    B, nh = q.shape[0], q.shape[1] // d
    g = nh // nkv
    out = torch.zeros(B, nh, d, dtype=torch.float64)
    mass = torch.zeros(B, nh, d, dtype=torch.float64)
    reach = torch.zeros(B, nh, 1, dtype=torch.float64)
    grown = None if weight is None else weight.double()
    for b in range(B):
        n, pos = int(lengths[b]), int(positions[b])
        if n < 0:
            continue
        bad = n >= table.shape[1] * S or not 0 <= pos < len(cos)
        if not bad:
            used = table[b, :n // S + 1].long()
            if 0 <= used[-1] < P:
                kp[used[-1], :, n % S] = rope32(k[b].float().view(nkv, d), cos[pos], sin[pos]).to(kp.dtype)
                vp[used[-1], :, n % S] = v[b].view(nkv, d)
            bad = bool(((used < 0) | (used >= P)).any())
        if bad:
            out[b] = math.nan
            continue
        qr = rope32(q[b].float().view(nh, d), cos[pos], sin[pos]).double()
        for h in range(nkv):
            kk, vv = (gather(t, table[b], h, n + 1, S).double() for t in (kp, vp))
            qh = qr[h * g:(h + 1) * g]
            p = torch.softmax(qh @ kk.t() / math.sqrt(d), -1)
            out[b, h * g:(h + 1) * g] = p @ vv
            mass[b, h * g:(h + 1) * g] = p @ vv.abs()
            reach[b, h * g:(h + 1) * g, 0] = (qh.abs() @ kk.abs().t()).amax(-1) / math.sqrt(d)
            if grown is not None:
                j = torch.arange(n + 1)
                pg = table[b].long()[j // S]
                grown[pg[-1], h, n % S] = 0.0
                grown[pg, h, j % S] += p.sum(0)
    return out.view(B, -1), mass.view(B, -1), reach.expand(-1, -1, d).reshape(B, -1), grown


def evict(kp, vp, weight, table, lengths, new_table, keep, recent):
    """The new lengths; the pages of new_table are filled in place."""
    P, nkv, S, d = kp.shape
    new_lengths = []
    src = [t.clone() for t in (kp, vp, weight)]
    for b, n in enumerate(lengths.tolist()):
        if n < 0 or n > table.shape[1] * S:
            new_lengths.append(-1)
            continue
        m = min(n, keep)
        new_lengths.append(m)
        for h in range(nkv):
            slots = list(range(n))
            if n > keep:
                w = gather(src[2], table[b], h, n, S).tolist()
                early = sorted(range(n - recent), key=lambda j: (0 if math.isnan(w[j]) else 1,
                                                                 0.0 if math.isnan(w[j]) else -w[j], j))
                slots = sorted(early[:keep - recent]) + list(range(n - recent, n))
            s, j = torch.tensor(slots, dtype=torch.long), torch.arange(m)
            for old, t in zip(src, (kp, vp, weight)):
                t[new_table[b].long()[j // S], h, j % S] = old[table[b].long()[s // S], h, s % S]
    return torch.tensor(new_lengths, dtype=torch.int32)


def attention_case(B_lens, nh, nkv, d, S, dtype, seed, weights=True, width=None, spare=3, angles=None):
    """Inputs of one attention call on the CPU; pages hold NaN wherever no token lies."""
    B = len(B_lens)
    P, table = pages_for([n + 1 for n in B_lens], S, seed, spare, width)
    kp = torch.full((P, nkv, S, d), math.nan, dtype=dtype)
    vp = torch.full((P, nkv, S, d), math.inf, dtype=dtype)
    weight = torch.full((P, nkv, S), math.nan) if weights else None
    for b, n in enumerate(B_lens):
        if n <= 0:
            continue
        j = torch.arange(n)
        pg = table[b].long()[j // S]
        kp[pg, :, j % S] = randn((n, nkv, d), seed + 10 * b + 1, dtype=dtype)
        vp[pg, :, j % S] = randn((n, nkv, d), seed + 10 * b + 2, dtype=dtype)
        if weights:
            weight[pg, :, j % S] = randn((n, nkv), seed + 10 * b + 3, dtype=torch.float32).abs()
    cos, sin = tables(angles or max(max(B_lens), 0) + 20, d)
    lengths = torch.tensor(B_lens, dtype=torch.int32)
    return dict(q=randn((B, nh * d), seed + 4, dtype=dtype), k=randn((B, nkv * d), seed + 5, dtype=dtype),
                v=randn((B, nkv * d), seed + 6, dtype=dtype), cos=cos, sin=sin, k_pages=kp, v_pages=vp, table=table,
                lengths=lengths, positions=(lengths.clamp(min=0) + 13).int(), weight=weight)
