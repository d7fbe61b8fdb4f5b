"""What is measured of the operators of batched decoding over a paged key-value
cache: appending tokens to the pages, the attention of one new token of every
sequence, eviction by accumulated attention weight, and the log probabilities of
tokens with their entropy and top alternatives.

With ``own`` false ``run`` computes them from elementary torch operations in 32
bits, rounded once; with ``own`` true it calls ``int4_hip``.  ``listed()`` gives the
fixed cases, ``draw(rng)`` further ones of the same ranges, ``prepare`` what a
program holds before the call, ``work`` the bytes and operations a pass cannot do
without and ``exact`` the result in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
MOST_BYTES = 5.5e8  # of the largest listed case


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one chat turn: one short sequence, the smallest call, latency alone
        dict(name="attention_1x100", kind="attention", B=1, L=100, ragged=False, nh=32, nkv=8, d=64, S=64,
             dtype="bf16", weights=False, idle=0),
        # a full decode batch of sequences of every length, two rows of it idle
        dict(name="attention_32_ragged_4k", kind="attention", B=32, L=4000, ragged=True, nh=32, nkv=8, d=64, S=16,
             dtype="bf16", weights=False, idle=2),
        # a batch whose cache will be evicted from: the weights are accumulated; wider heads, fp16
        dict(name="attention_16x3001_weights", kind="attention", B=16, L=3001, ragged=False, nh=32, nkv=8, d=128,
             S=64, dtype="fp16", weights=True, idle=0),
        # one document at the end of a long context: few rows, all of the chip on one sequence
        dict(name="attention_1x131000", kind="attention", B=1, L=131000, ragged=False, nh=32, nkv=8, d=128, S=64,
             dtype="bf16", weights=False, idle=0),
        # the accumulated weights of a long sequence, many query heads on few key heads
        dict(name="attention_3x20000_weights", kind="attention", B=3, L=20000, ragged=True, nh=20, nkv=2, d=128,
             S=128, dtype="bf16", weights=True, idle=0),
        # a prompt put into the cache after its prefill
        dict(name="append_prompt_7999", kind="append", B=1, T=7999, nkv=8, d=128, S=64, dtype="bf16", weights=True),
        # two ragged chunks of prompts, small heads, small pages, fp16
        dict(name="append_chunk_300", kind="append", B=2, T=300, nkv=8, d=64, S=16, dtype="fp16", weights=False),
        # a sequence over its budget by a page
        dict(name="evict_1x576", kind="evict", B=1, L=576, ragged=False, keep=512, recent=64, nkv=8, d=64, S=64,
             dtype="bf16"),
        # a batch of long prompts cut to an eighth
        dict(name="evict_4x32768", kind="evict", B=4, L=32768, ragged=True, keep=4096, recent=500, nkv=8, d=128, S=64,
             dtype="fp16"),
        # a decode batch's next tokens with five alternatives
        dict(name="logprobs_8_top5", kind="logprobs", R=8, V=128256, top=5, dtype="bf16"),
        # a prompt scored against its own tokens, with what an evaluation keeps of each row
        dict(name="logprobs_500_top20", kind="logprobs", R=500, V=128256, top=20, dtype="bf16"),
        # a small odd vocabulary, fp32 logits, no alternatives
        dict(name="logprobs_1000_32001", kind="logprobs", R=1000, V=32001, top=0, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 64), (32, 8, 128), (8, 2, 64), (16, 16, 64), (20, 2, 128), (6, 1, 128), (24, 1, 64), (12, 4, 128)]


def draw(rng):
    """A case of the listed ones' ranges, made smaller until it costs no more than the largest of them."""
    kind = rng.choice(["attention", "attention", "append", "evict", "logprobs"])
    nh, nkv, d = rng.choice(HEADS)
    S, dtype = rng.choice([16, 32, 64, 128, 256]), rng.choice(["bf16", "fp16"])
    if kind == "attention":
        B = _log(rng, 1, 96)
        c = dict(kind=kind, B=B, L=_log(rng, 1, 131072), ragged=rng.random() < 0.6, nh=nh, nkv=nkv, d=d, S=S,
                 dtype=dtype, weights=rng.random() < 0.4, idle=rng.randint(0, B // 8))
        small = "L"
    elif kind == "append":
        B = _log(rng, 1, 64)
        c = dict(kind=kind, B=B, T=max(B, _log(rng, 1, 16384)), nkv=nkv, d=d, S=S, dtype=dtype,
                 weights=rng.random() < 0.5)
        small = "T"
    elif kind == "evict":
        L = _log(rng, 64, 131072)
        keep = max(1, int(L * rng.uniform(0.05, 0.98)))
        c = dict(kind=kind, B=_log(rng, 1, 48), L=L, ragged=rng.random() < 0.5, keep=keep,
                 recent=int(keep * rng.choice([0.0, 0.1, 0.5, 1.0])), nkv=nkv, d=d, S=S, dtype=dtype)
        small = "B"
    else:
        c = dict(kind=kind, R=_log(rng, 1, 2048), V=rng.choice([128256, 32001, _log(rng, 100, 200000)]),
                 top=rng.choice([0, 1, 2, 5, 8, 20, 32, 64]), dtype=rng.choice(["bf16", "fp16", "fp32"]))
        small = "R"
    # the padded plain form also has to fit: rows times the longest length
    while work(c)["bytes"] > MOST_BYTES or ("L" in c and c["B"] * c["L"] * c["nkv"] * c["d"] * 4 > 3 * MOST_BYTES):
        if c[small] > 1:
            c[small] //= 2
        else:
            c["L"] //= 2
            c["keep"] = max(1, c["keep"] // 2)
            c["recent"] = min(c["recent"], c["keep"])
        if kind == "append":
            c["B"] = min(c["B"], c["T"])
    return c


def _lens(c):
    """Tokens already in the cache of every row: of the case alone, spread over 1..L where ragged; -1 for idle rows."""
    B, L = c["B"], c["L"]
    n = [max(1, int(L * (((b + 1) * 0.6180339887) % 1.0))) if c["ragged"] and b else L for b in range(B)]
    for i in range(c.get("idle", 0)):
        n[B - 1 - 3 * i if B - 1 - 3 * i > 0 else B - 1] = -1
    return n


def _chunks(c):
    """Tokens of every row of an append, and the slot its first one goes to."""
    B, T = c["B"], c["T"]
    n = [T // B + (1 if b < T % B else 0) for b in range(B)]
    return n, [(37 * b) % 200 for b in range(B)]


# ------------------------------------------------------------------ inputs
def _tables(n, d):
    ang = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * (
        1.0 / 500000.0 ** (torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d))[None, :]
    return ang.cos().float(), ang.sin().float()


def _pool(lens, S, g, reserve=1):
    """(pages in the pool, table [B, W] int32): pages in random order, -1 where a row has none."""
    need = [max(1, -(-n // S)) for n in lens]
    B, W = len(lens), max(need)
    ids = torch.randperm(sum(need) + reserve, generator=g, device=DEV).to(torch.int32)
    per = torch.tensor(need, device=DEV)
    used = torch.arange(W, device=DEV)[None, :] < per[:, None]
    start = torch.cumsum(per, 0) - per
    at = (start[:, None] + torch.arange(W, device=DEV)[None, :]).clamp_(max=len(ids) - 1)
    return len(ids), torch.where(used, ids[at], torch.full_like(ids[at], -1)).contiguous()


def _randn(shape, dtype, g, scale=1.0):
    """Normal values, made in pieces so that the 32-bit form of a large tensor never exists."""
    t = torch.empty(shape, dtype=dtype, device=DEV)
    flat = t.view(-1)
    for i in range(0, flat.numel(), 1 << 26):
        part = flat[i:i + (1 << 26)]
        part.copy_(torch.randn(part.numel(), generator=g, device=DEV) * scale)
    return t


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "logprobs":
        R, V = c["R"], c["V"]
        logits = _randn((R, V), dt, g, 2.5)
        # a few tokens that the model favours, as in real text
        top = torch.randint(0, V // 8, (R, 8), generator=g, device=DEV) + torch.arange(8, device=DEV) * (V // 8)
        logits.scatter_add_(1, top, (torch.rand((R, 8), generator=g, device=DEV) * 14).to(dt))
        return dict(kind="logprobs", logits=logits, tokens=top[:, 0].contiguous(), top=c["top"])
    nkv, d, S = c["nkv"], c["d"], c["S"]
    s = dict(kind=c["kind"])
    if c["kind"] == "append":
        n, first = _chunks(c)
        P, s["table"] = _pool([a + b for a, b in zip(n, first)], S, g)
        count = torch.tensor(n, device=DEV)
        s["rows"] = torch.repeat_interleave(torch.arange(c["B"], device=DEV), count).to(torch.int32)
        start = torch.cumsum(count, 0) - count
        local = torch.arange(c["T"], device=DEV) - start[s["rows"].long()]
        s["slots"] = (local + torch.tensor(first, device=DEV)[s["rows"].long()]).to(torch.int32)
        s["positions"] = s["slots"] + 11  # eleven tokens were evicted before
        s["cos"], s["sin"] = _tables(max(a + b for a, b in zip(n, first)) + 12, d)
        s["k"], s["v"] = (_randn((c["T"], nkv * d), dt, g) for _ in range(2))
        weights = c["weights"]
    elif c["kind"] == "attention":
        n = _lens(c)
        P, s["table"] = _pool([x + 1 for x in n], S, g)
        s["lengths"] = torch.tensor(n, dtype=torch.int32, device=DEV)
        s["positions"] = s["lengths"].clamp(min=0) + 11
        s["cos"], s["sin"] = _tables(max(n) + 13, d)
        s["q"] = _randn((c["B"], c["nh"] * d), dt, g)
        s["k"], s["v"] = (_randn((c["B"], nkv * d), dt, g) for _ in range(2))
        weights = c["weights"]
    else:
        n = _lens(c)
        both, table = _pool(n + [min(x, c["keep"]) for x in n], S, g)
        P, B = both, c["B"]
        s["table"], s["new_table"] = table[:B].contiguous(), table[B:, :-(-c["keep"] // S)].contiguous()
        s["lengths"] = torch.tensor(n, dtype=torch.int32, device=DEV)
        s["keep"], s["recent"] = c["keep"], c["recent"]
        weights = True
    s["k_pages"], s["v_pages"] = (_randn((P, nkv, S, d), dt, g) for _ in range(2))
    if weights:
        # a few heavy tokens, many light ones, some never looked at
        w = torch.randn((P, nkv, S), generator=g, device=DEV).mul_(2.5).exp_().mul_(1e-3)
        s["weight"] = w.masked_fill_(torch.rand((P, nkv, S), generator=g, device=DEV) < 0.02, 0.0)
    else:
        s["weight"] = None
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    s = state
    if own:
        return _own(s)
    return {"logprobs": _logprobs, "append": _append, "attention": _attention, "evict": _evict}[s["kind"]](s)


def _outputs(s, **more):
    out = dict(more, k_pages=s["k_pages"], v_pages=s["v_pages"])
    if s["weight"] is not None:
        out["weight"] = s["weight"]
    return out


def _package():
    import sys
    from pathlib import Path

    at = str(Path.cwd() / "itmo-final-project_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import int4_hip

    return int4_hip


def _own(s):
    op = _package()
    if s["kind"] == "logprobs":
        r = op.token_logprobs(s["logits"], s["tokens"], top=s["top"])
        return dict(logprob=r.logprob, entropy=r.entropy, top_logprob=r.top_logprob, top_token=r.top_token)
    if s["kind"] == "append":
        op.paged_append(s["k"], s["v"], s["cos"], s["sin"], s["k_pages"], s["v_pages"], s["table"], s["rows"],
                        s["slots"], s["positions"], weight=s["weight"])
        return _outputs(s)
    if s["kind"] == "attention":
        out = op.paged_attention(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_pages"], s["v_pages"], s["table"],
                                 s["lengths"], s["positions"], weight=s["weight"])
        return _outputs(s, out=out)
    n = op.paged_evict(s["k_pages"], s["v_pages"], s["weight"], s["table"], s["lengths"], s["new_table"], s["keep"],
                       s["recent"])
    return _outputs(s, lengths=n)


def _rope(x, cos, sin):
    """x [T, heads, d] fp32, cos and sin [T, d / 2]: the two halves of d rotated."""
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cos[:, None, :], sin[:, None, :]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _append(s):
    nkv, S, d = s["k_pages"].shape[1:]
    T, dt, pos = s["k"].shape[0], s["k"].dtype, s["positions"].long()
    slots = s["slots"].long()
    page = s["table"].long()[s["rows"].long(), slots // S]
    at = slots % S
    k = _rope(s["k"].float().view(T, nkv, d), s["cos"][pos], s["sin"][pos])
    s["k_pages"][page, :, at] = k.to(dt)
    s["v_pages"][page, :, at] = s["v"].view(T, nkv, d)
    if s["weight"] is not None:
        s["weight"][page, :, at] = 0.0
    return _outputs(s)


def _attention(s):
    P, nkv, S, d = s["k_pages"].shape
    B, dt = s["q"].shape[0], s["q"].dtype
    g = s["q"].shape[1] // (nkv * d)
    n, pos, dev = s["lengths"].long(), s["positions"].long(), s["q"].device
    live = n >= 0
    last = n.clamp(min=0)
    cos, sin = s["cos"][pos], s["sin"][pos]
    table = s["table"].long().clamp(min=0)
    # the new token; an idle row keeps what its first slot holds
    page, at = table.gather(1, (last // S)[:, None])[:, 0], last % S
    k = _rope(s["k"].float().view(B, nkv, d), cos, sin).to(dt)
    keep = live[:, None, None]
    s["k_pages"][page, :, at] = torch.where(keep, k, s["k_pages"][page, :, at])
    s["v_pages"][page, :, at] = torch.where(keep, s["v"].view(B, nkv, d), s["v_pages"][page, :, at])
    # every row's pages side by side: [B, nkv, W * S, d]
    cap = table.shape[1] * S
    seen = (torch.arange(cap, device=dev)[None, :] <= n[:, None])[:, None, :, None]
    kk = s["k_pages"][table].transpose(1, 2).reshape(B, nkv, cap, d).float()
    vv = s["v_pages"][table].transpose(1, 2).reshape(B, nkv, cap, d).float().masked_fill_(~seen, 0.0)
    q = _rope(s["q"].float().view(B, nkv * g, d), cos, sin).view(B, nkv, g, d)
    x = torch.matmul(kk, q.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))  # [B, nkv, cap, g]
    x = x.masked_fill_(~seen, -math.inf)
    top = x.amax(2, keepdim=True)
    e = torch.exp(x - torch.where(live[:, None, None, None], top, torch.zeros_like(top)))
    p = e / e.sum(2, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p.transpose(2, 3).contiguous(), vv).to(dt).view(B, nkv * g * d)
    if s["weight"] is not None:
        w = s["weight"]
        w[page, :, at] = torch.where(live[:, None], torch.zeros_like(w[page, :, at]), w[page, :, at])
        slot = torch.arange(cap, device=dev)
        to = (table[:, slot // S][:, None, :] * nkv + torch.arange(nkv, device=dev)[None, :, None]) * S + slot % S
        w.view(-1).scatter_add_(0, to.reshape(-1), p.sum(3).reshape(-1))  # what is not seen adds zeros
    return _outputs(s, out=out)


def _evict(s):
    P, nkv, S, d = s["k_pages"].shape
    n, keep, recent, dev = s["lengths"].long(), s["keep"], s["recent"], s["lengths"].device
    B, cap = n.shape[0], s["table"].shape[1] * S
    table, new = s["table"].long().clamp(min=0), s["new_table"].long().clamp(min=0)
    slot, heads = torch.arange(cap, device=dev), torch.arange(nkv, device=dev)[None, :, None]
    flat = (table[:, slot // S][:, None, :] * nkv + heads) * S + slot % S  # [B, nkv, cap]
    w = s["weight"].view(-1)[flat]
    # rank by: recent tokens, then weights, then nothing; a stable sort puts the lowest slot first among equals
    inside, late = slot[None, :] < n[:, None], slot[None, :] >= (n - recent)[:, None]
    w = w.masked_fill(late[:, None, :], math.inf).masked_fill(~inside[:, None, :], -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :min(keep, cap)]
    m = torch.minimum(n, torch.full_like(n, keep))
    there = torch.arange(order.shape[-1], device=dev)[None, :] < m[:, None]  # [B, keep]
    order = torch.sort(order.masked_fill(~there[:, None, :], cap), dim=-1).values.clamp(max=cap - 1)
    src = flat.gather(2, order)
    j = torch.arange(order.shape[-1], device=dev)
    dst = (new[:, j // S][:, None, :] * nkv + heads) * S + j % S
    for name in ("k_pages", "v_pages", "weight"):
        t = s[name].view(P * nkv * S, -1)
        ok = there[:, None, :, None]
        t[dst] = torch.where(ok, t[src], t[dst])
    return _outputs(s, lengths=m.to(torch.int32))


def _logprobs(s):
    x, top, V = s["logits"].float(), s["top"], s["logits"].shape[1]
    m = x.amax(1, keepdim=True)
    y = x - m
    e = torch.exp(y)
    z = e.sum(1, keepdim=True)
    logz = torch.log(z)
    entropy = logz[:, 0] - (e * y).sum(1) / z[:, 0]
    logprob = (y.gather(1, s["tokens"][:, None]) - logz)[:, 0]
    # the largest values, the lowest index first among equals: one whole number orders both
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = order * (1 << 32) + (V - 1 - torch.arange(V, device=x.device))
    token = torch.topk(key, top, dim=1).indices
    return dict(logprob=logprob, entropy=entropy, top_logprob=y.gather(1, token) - logz, top_token=token)


# ------------------------------------------------------------------ floors
def work(case):
    c = case
    e = SIZE[c["dtype"]]
    if c["kind"] == "logprobs":
        R, V, top = c["R"], c["V"], c["top"]
        return {"bytes": R * V * e + R * (8 + 4 + 4 + 12 * top), "flops": 5 * R * V}
    nkv, d = c["nkv"], c["d"]
    if c["kind"] == "append":
        T = c["T"]
        return {"bytes": T * (4 * nkv * d * e + 4 * d + 12 + (4 * nkv if c["weights"] else 0)),
                "flops": 3 * T * nkv * d}
    n = _lens(c)
    if c["kind"] == "attention":
        live = [x + 1 for x in n if x >= 0]
        old, rows = sum(live) - len(live), len(live)
        b = old * nkv * d * 2 * e  # the cache
        b += rows * (2 * c["nh"] * d * e + 4 * nkv * d * e + 4 * d)  # q, out; the new key and value in and out; angles
        b += (sum(live) + old) * nkv * 4 if c["weights"] else 0
        b += sum(-(-x // c["S"]) for x in live) * 4 + 8 * c["B"]
        return {"bytes": b, "flops": 4 * sum(live) * c["nh"] * d}
    m = sum(min(x, c["keep"]) for x in n)
    scored = sum(x for x in n if x > c["keep"]) if c["recent"] < c["keep"] else 0
    return {"bytes": scored * nkv * 4 + 2 * m * nkv * (2 * d * e + 4), "flops": scored * nkv}


# ------------------------------------------------------------------ 64 bits
def _rotated(x, angle_cos, angle_sin):
    x, c, s = x.double(), angle_cos.double(), angle_sin.double()
    half = x.shape[-1] // 2
    first, second = x[..., :half], x[..., half:]
    return torch.cat([first * c - second * s, first * s + second * c], dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "logprobs":
        return _exact_logprobs(s)
    w = None if s["weight"] is None else s["weight"].double()
    if s["kind"] == "evict":
        return _exact_evict(s, w)
    kp, vp, table = s["k_pages"], s["v_pages"], s["table"].cpu().tolist()
    S, d, nkv = kp.shape[2], kp.shape[3], kp.shape[1]
    out = None
    ko, vo = kp.double(), vp.double()
    if s["kind"] == "append":
        rows, slots, where = (s[k].cpu().tolist() for k in ("rows", "slots", "positions"))
        page = torch.tensor([table[r][t // S] for r, t in zip(rows, slots)], device=DEV)
        at = torch.tensor([t % S for t in slots], device=DEV)
        angle = torch.tensor(where, device=DEV)
        ko[page, :, at] = _rotated(s["k"].view(-1, nkv, d), s["cos"][angle][:, None], s["sin"][angle][:, None])
        vo[page, :, at] = s["v"].view(-1, nkv, d).double()
        if w is not None:
            w[page, :, at] = 0.0
    else:
        lens, where = s["lengths"].cpu().tolist(), s["positions"].cpu().tolist()
        q = s["q"].view(len(lens), nkv, -1, d)
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(lens):
            if n < 0:
                continue
            c, t = s["cos"][where[b]], s["sin"][where[b]]
            pages = torch.tensor(table[b][:n // S + 1], device=DEV)
            key = _rotated(s["k"][b].view(nkv, d), c, t)
            kp[pages[-1], :, n % S] = key.to(kp.dtype)
            vp[pages[-1], :, n % S] = s["v"][b].view(nkv, d)
            ko[pages[-1], :, n % S] = key
            vo[pages[-1], :, n % S] = s["v"][b].view(nkv, d).double()
            query = _rotated(q[b], c, t)
            for h in range(nkv):
                keys = kp[pages, h].reshape(-1, d)[:n + 1].double()
                p = torch.softmax(query[h] @ keys.t().contiguous() / math.sqrt(d), dim=-1)
                out[b, h] = p @ vp[pages, h].reshape(-1, d)[:n + 1].double()
                if w is not None:
                    full = torch.zeros(len(pages) * S, dtype=torch.float64, device=DEV)
                    full[:n + 1] = p.sum(0)
                    w[pages[-1], h, n % S] = 0.0
                    w[pages, h] += full.view(-1, S)
        out = out.view(len(lens), -1)
    got = dict(k_pages=ko, v_pages=vo)
    if out is not None:
        got["out"] = out
    if w is not None:
        got["weight"] = w
    return got


def _exact_evict(s, w):
    kp, vp, wt = s["k_pages"].clone(), s["v_pages"].clone(), s["weight"].clone()
    S, nkv, keep = kp.shape[2], kp.shape[1], s["keep"]
    lens, table, new = (s[k].cpu().tolist() for k in ("lengths", "table", "new_table"))
    for b, n in enumerate(lens):
        m, late = min(n, keep), min(s["recent"], keep, n)
        old = torch.tensor(table[b][:-(-n // S)], device=DEV)
        to = torch.tensor(new[b][:-(-m // S)], device=DEV)
        for h in range(nkv):
            mass = w[old, h].reshape(-1)[:n]
            if n > keep:
                # the threshold, then as many of its equals as are left to take, from the front
                early = mass[:n - late]
                want = keep - late
                if want:
                    edge = torch.sort(early).values[-want]
                    more, same = early > edge, early == edge
                    take = more | (same & (torch.cumsum(same, 0) <= want - more.sum()))
                else:
                    take = torch.zeros_like(early, dtype=torch.bool)
                kept = torch.cat([take.nonzero()[:, 0], torch.arange(n - late, n, device=DEV)])
            else:
                kept = torch.arange(n, device=DEV)
            j = torch.arange(m, device=DEV)
            for src, dst in ((s["k_pages"], kp), (s["v_pages"], vp), (s["weight"], wt)):
                dst[to[j // S], h, j % S] = src[old[kept // S], h, kept % S]
    return dict(lengths=None, k_pages=kp.double(), v_pages=vp.double(), weight=wt.double())


def _exact_logprobs(s):
    parts = []
    for rows, tokens in zip(s["logits"].split(256), s["tokens"].split(256)):
        x = rows.double()
        logp = torch.log_softmax(x, dim=-1)
        entropy = -(logp.exp() * logp).sum(-1)
        best = torch.sort(logp, dim=-1, descending=True).values[:, :s["top"]]
        parts.append((logp.gather(1, tokens[:, None])[:, 0], entropy, best))
    logprob, entropy, best = (torch.cat(p) for p in zip(*parts))
    return dict(logprob=logprob, entropy=entropy, top_logprob=best, top_token=None)
