"""Plain 64-bit statement of the 8-bit paged cache's operators and of the verification
of drafts, row by row on the CPU, and the inputs their tests share."""
from __future__ import annotations

import bisect
import math

import torch

from _paged_ref import pages_for, tables
from _synth import randn

NAN = float("nan")
CODES = [torch.int8, torch.float8_e4m3fn]
MOST = {torch.int8: 127, torch.float8_e4m3fn: 448}
TINY = 2.0 ** -126


def _codes(kind):
    """(values in order, their codes): what the codes that are numbers stand for, one code each."""
    every = torch.arange(256, dtype=torch.int16).to(torch.uint8)
    x = every.view(kind).double()
    table = {}
    for c, v in zip(every.tolist(), x.tolist()):
        if v == v and abs(v) <= MOST[kind]:
            table.setdefault(v, c)
    values = sorted(table)
    return values, [table[v] for v in values]


_TABLE = {kind: _codes(kind) for kind in CODES}


def nearest(y, kind):
    """The value that a code stands for nearest to the number ``y``, of two the one with an even code."""
    values, codes = _TABLE[kind]
    i = bisect.bisect_left(values, y)
    if i == 0 or i == len(values):
        return values[min(i, len(values) - 1)]
    lo, hi = values[i - 1], values[i]
    if y - lo != hi - y:
        return lo if y - lo < hi - y else hi
    return lo if codes[i - 1] % 2 == 0 else hi


def quantise(x, s, kind):
    """Values in units of the scale ``s`` for the tensor ``x`` of 64 bits."""
    if not s > 0:  # zero, or NaN
        return torch.zeros_like(x)
    y = x / torch.full_like(x, s)
    return torch.tensor([nearest(v, kind) for v in y.flatten().tolist()], dtype=torch.float64).view(x.shape)


def rotate(x, cos, sin):
    """x [heads, d] in 64 bits at one position's angles [d / 2]."""
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cos.double(), sin.double()
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def new_key(k, cos, sin, pos, nkv, d):
    x = k.double().view(nkv, d)
    return rotate(x, cos[pos], sin[pos]) if 0 <= pos < len(cos) else torch.full_like(x, NAN)


def append(k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths, offsets, positions, **_):
    """All in place: the pages hold codes, of which those that are 0 may come out with either sign."""
    P, nkv, S, d = k_pages.shape
    block = S // k_scale.shape[2]
    for b in range(len(lengths)):
        n, o0, o1 = int(lengths[b]), int(offsets[b]), int(offsets[b + 1])
        if n < 0 or o1 <= o0 or n + o1 - o0 > table.shape[1] * S:
            continue
        for j in range(n // block, (n + o1 - o0 - 1) // block + 1):
            lo, hi = max(n, j * block), min(n + o1 - o0, (j + 1) * block)
            page = int(table[b, j * block // S])
            if not 0 <= page < P:
                continue
            t = range(o0 + lo - n, o0 + hi - n)
            keys = torch.stack([new_key(k[i], cos, sin, int(positions[i]), nkv, d) for i in t])
            vals = torch.stack([v[i].double().view(nkv, d) for i in t])
            at = j * block % S
            for x, pages, scales in ((keys, k_pages, k_scale), (vals, v_pages, v_scale)):
                kind = pages.dtype
                for h in range(nkv):
                    a = float(x[:, h].abs().max())
                    old = 0.0 if lo == j * block else float(scales[page, h, at // block])
                    if not math.isfinite(float(x[:, h].abs().sum())) or old != old:
                        s = NAN
                    elif old > 0:
                        s = old
                        while a > MOST[kind] * s:
                            s *= 2
                        if s > old:
                            was = pages[page, h, at:at + block].double()  # (what is new is written over)
                            new = quantise(was * old, s, kind)
                            new = torch.where(was.isnan(), was, new)
                            pages[page, h, at:at + block] = new.float().to(kind)
                    else:
                        s = max(float(torch.tensor(a / MOST[kind], dtype=torch.float64).float()), TINY) if a > 0 else 0.0
                    scales[page, h, at // block] = s
                    pages[page, h, at + lo - j * block:at + hi - j * block] = quantise(x[:, h], s, kind).float().to(kind)


def values(pages, scales, row, n):
    """Slots 0..n-1 of a table row, [n, kv_heads, d] in 64 bits; NaN where there is no page, or a code of NaN."""
    P, nkv, S, d = pages.shape
    block = S // scales.shape[2]
    out = torch.full((n, nkv, d), NAN, dtype=torch.float64)
    for i in range(0, n, 8):
        page = int(row[i // S])
        if 0 <= page < P:
            m, s = min(8, n - i), scales[page, :, i % S // block].double()
            out[i:i + m] = (pages[page, :, i % S:i % S + m].double() * s[:, None, None]).transpose(0, 1)
    return out


def read(k_pages, v_pages, k_scale, v_scale, table, starts, offsets, tokens, dtype):
    P, nkv, S, d = k_pages.shape
    out = torch.zeros(2, tokens, nkv, d, dtype=torch.float64)
    for b in range(len(starts)):
        n, o0, o1 = int(starts[b]), int(offsets[b]), int(offsets[b + 1])
        if n < 0 or o1 <= o0:
            continue
        most = min(n + o1 - o0, table.shape[1] * S)
        out[:, o0:o1] = NAN
        for x, pages, scales in ((out[0], k_pages, k_scale), (out[1], v_pages, v_scale)):
            x[o0:o0 + max(most - n, 0)] = values(pages, scales, table[b], most)[n:]
    return tuple(x.float().to(dtype).flatten(1) for x in out)


def attention(q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths, offsets, positions, window=None,
              sinks=0, **_):
    """(out, p @ |v|, the largest sum |q||k| / sqrt(d) that a token's head meets) in 64 bits; the cache is updated in
    place."""
    append(k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths, offsets, positions)
    P, nkv, S, d = k_pages.shape
    T, nh = q.shape[0], q.shape[1] // d
    out, mass = (torch.zeros(T, nh, d, dtype=torch.float64) for _ in range(2))
    reach = torch.zeros(T, nh, 1, dtype=torch.float64)
    for b in range(len(lengths)):
        n, o0, o1 = int(lengths[b]), int(offsets[b]), int(offsets[b + 1])
        if n < 0:
            continue
        if n + o1 - o0 > table.shape[1] * S:
            out[o0:o1] = NAN
            continue
        kk, vv = (values(x, s, table[b], n + o1 - o0) for x, s in ((k_pages, k_scale), (v_pages, v_scale)))
        scale = values(torch.ones_like(v_pages), v_scale, table[b], n + o1 - o0)[..., 0]
        for t in range(o0, o1):
            i = n + t - o0
            j = torch.arange(i + 1)
            seen = j if window is None else j[(j > i - window) | (j < sinks)]
            pos = int(positions[t])
            x = q[t].double().view(nh, d)
            x = rotate(x, cos[pos], sin[pos]) if 0 <= pos < len(cos) else torch.full_like(x, NAN)
            for h in range(nkv):
                key, val, heads = kk[seen, h], vv[seen, h], slice(h * nh // nkv, (h + 1) * nh // nkv)
                p = torch.softmax(key @ x[heads].T / math.sqrt(d), 0).T
                # (a probability that fp32 cannot have, 2^-118 of the largest with the reference 2^8 behind, is lost: the
                # tolerance, 2^-21 of the mass or more, is to hold n 2^-110 of the largest value)
                # (weights, probability times scale, enter as two numbers of 11 bits each, whose smallest step is 2^-24:
                # with the column's largest raised past 2^10, they are within 2^-35 of the largest at worst, 2^-14 of
                # that 2^-21)
                step = scale[seen, h]
                sums = (val / step[:, None]).nan_to_num().abs().sum(0)
                out[t, heads] = p @ val
                mass[t, heads] = (p @ val.abs() + len(seen) * 2.0 ** -89 * val.nan_to_num().abs().max()
                                  + 2.0 ** -14 * (p * step).nan_to_num().amax(1, True) * sums)
                reach[t, heads] = (x[heads].abs() @ key.abs().T).amax(1, True) / math.sqrt(d)
                out[t, heads][~x[heads].isfinite().all(1) | ~key.isfinite().all()] = NAN
    return out.flatten(1), mass.flatten(1), reach.expand(-1, -1, d).flatten(1)


def cache(kind, P, nkv, S, d, block, seed):
    """Pages as a program has left them, and their scales: codes of normal values."""
    r = {}
    for i, n in enumerate("kv"):
        x = randn((P, nkv, S, d), seed=seed + i).float() * 0.3 * MOST[kind]
        x = x.clamp(-MOST[kind], MOST[kind])
        r[n + "_pages"] = (x.round() if kind == torch.int8 else x).to(kind)
        r[n + "_scale"] = (randn((P, nkv, S // block), seed=seed + 7 + i).float().abs() + 0.1) / MOST[kind]
    return r


def case(lens, new, nh, nkv, d, S, block, kind, dtype, seed=0, width=None, shift=11, angles=None, **more):
    """Inputs of a call: rows of ``lens`` slots (-1: idle) with ``new`` new tokens each, by name."""
    P, table = pages_for([max(n, 0) + m for n, m in zip(lens, new)], S, seed, width=width)
    offsets = [sum(new[:b]) for b in range(len(new) + 1)]
    T = offsets[-1]
    positions = [max(n, 0) + j + shift for n, m in zip(lens, new) for j in range(m)]
    cos, sin = tables(angles or max([shift] + positions) + 1, d)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return dict(q=randn((T, nh * d), seed=seed + 3, dtype=dtype), k=randn((T, nkv * d), seed=seed + 4, dtype=dtype),
                v=randn((T, nkv * d), seed=seed + 5, dtype=dtype), cos=cos, sin=sin,
                **cache(kind, P, nkv, S, d, block, seed + 20), table=table, lengths=i32(lens), offsets=i32(offsets),
                positions=i32(positions), **more)


def verify(target, draft, tokens, accept, sample, counts=None):
    B, K, V = tokens.shape[0], tokens.shape[1], target.shape[2]
    accepted, token = [], []
    for b in range(B):
        n = K if counts is None else int(counts[b])
        if not 0 <= n <= K:
            accepted.append(-1), token.append(-1)
            continue
        p = target[b].double()
        r = 0
        while r < n:
            x = int(tokens[b, r])
            q = 1.0 if draft is None else float(draft[b, r, x]) if 0 <= x < V else 0.0
            if not (0 <= x < V and float(accept[b, r]) * q < float(p[r, x])):
                break
            r += 1
        w = p[r].clone()
        if r < n:
            if draft is not None:
                w = w - draft[b, r].double()
            elif 0 <= int(tokens[b, r]) < V:
                w[int(tokens[b, r])] -= 1.0
        w = w.clamp(min=0)
        if float(w.sum()) == 0.0:
            w = p[r].clamp(min=0)
        total = float(w.sum())
        accepted.append(r)
        if not (math.isfinite(total) and total > 0):
            token.append(-1)
            continue
        upto, aim, hit = 0.0, float(sample[b]) * math.fsum(w.tolist()), -1
        for i, x in enumerate(w.tolist()):
            upto += x
            if x > 0:
                hit = i
                if upto > aim:
                    break
        token.append(hit)
    return torch.tensor(accepted), torch.tensor(token)
