"""What is measured of the operators of batched decoding over a paged cache held in 8
bits: tokens quantised as they are written and read back, attention of a few new
tokens of every row over such a cache (all of it, or a sliding window and a few first
tokens), and the verification of drafted tokens.

With ``own`` false ``run`` computes them from elementary torch operations, in 32 bits
(64 where a value next to a border of the quantisation, or a long sum, needs them);
with ``own`` true it calls ``int4_hip``.  ``listed()`` gives the fixed cases,
``draw(rng)`` further ones of the same ranges, ``prepare`` what a program holds before
the call, ``work`` the bytes and operations a pass cannot do without and ``exact`` the
result in 64 bits.
"""
from __future__ import annotations

import math
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127, "e4m3": 448}  # of a code's magnitudes
SMALLEST_SCALE = 2.0 ** -126
MOST_BYTES, MOST_FLOPS = 3.7e8, 1.65e10  # of the largest listed cases


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one chat turn: one short sequence, the smallest call, latency alone
        dict(name="attention_1x100", kind="attention", B=1, L=100, ragged=False, T=1, nh=32, nkv=8, d=64, S=64,
             block=16, codes="int8", dtype="bf16", window=0, sinks=0, idle=0),
        # a full decode batch of sequences of every length, two rows of it idle
        dict(name="attention_32_ragged_4k", kind="attention", B=32, L=4000, ragged=True, T=1, nh=32, nkv=8, d=64, S=16,
             block=16, codes="e4m3", dtype="bf16", window=0, sinks=0, idle=2),
        # one document at the end of a long context: all of the chip on one sequence
        dict(name="attention_1x131000", kind="attention", B=1, L=131000, ragged=False, T=1, nh=32, nkv=8, d=128, S=64,
             block=32, codes="int8", dtype="bf16", window=0, sinks=0, idle=0),
        # long conversations of which every token sees the last 1000 and the first 4
        dict(name="attention_24x20000_window", kind="attention", B=24, L=20000, ragged=True, T=1, nh=32, nkv=8, d=128,
             S=64, block=64, codes="e4m3", dtype="fp16", window=1000, sinks=4, idle=0),
        # a speculative step: up to five drafted tokens a row
        dict(name="attention_16x3001_drafts5", kind="attention", B=16, L=3001, ragged=True, T=5, nh=32, nkv=8, d=128,
             S=64, block=32, codes="int8", dtype="fp16", window=0, sinks=0, idle=1),
        # a prompt at once
        dict(name="attention_prompt_2000", kind="attention", B=1, L=2000, ragged=False, T=2000, nh=32, nkv=8,
             d=64, S=64, block=64, codes="e4m3", dtype="bf16", window=0, sinks=0, idle=0),
        # a decode step's tokens, one a row, each into a block that holds some
        dict(name="write_32x1", kind="write", B=32, T=32, nkv=8, d=64, S=64, block=16, codes="int8", dtype="bf16",
             out="bf16"),
        # a prompt put into the cache
        dict(name="write_prompt_7999", kind="write", B=1, T=7999, nkv=8, d=128, S=64, block=32, codes="e4m3",
             dtype="bf16", out="bf16"),
        # a short shared prefix read back
        dict(name="read_1x300", kind="read", B=1, T=300, nkv=8, d=64, S=64, block=16, codes="int8", dtype="bf16",
             out="bf16"),
        # long rows read back, for a program that attends in its own way
        dict(name="read_5_of_60000", kind="read", B=5, T=60000, nkv=8, d=128, S=128, block=64, codes="e4m3",
             dtype="fp16", out="fp16"),
        # one sequence's four drafts
        dict(name="verify_1x4", kind="verify", B=1, K=4, V=128256, dtype="fp32", drafted=True, ragged=False),
        # a batch's, of different numbers of drafts
        dict(name="verify_48x5", kind="verify", B=48, K=5, V=128256, dtype="fp32", drafted=True, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 64), (32, 8, 128), (8, 2, 64), (16, 16, 64), (20, 2, 128), (6, 1, 128), (24, 1, 64), (12, 4, 128)]


def draw(rng):
    """A case of the listed ones' ranges, made smaller until it costs no more than the largest of them."""
    kind = rng.choice(["attention", "attention", "attention", "write", "read", "verify"])
    nh, nkv, d = rng.choice(HEADS)
    S = rng.choice([16, 32, 64, 128, 256])
    c = dict(kind=kind, B=_log(rng, 1, 64))
    if kind == "verify":
        c |= dict(K=rng.choice([1, 2, 3, 4, 5, 8]), V=rng.choice([128256, 32001, _log(rng, 100, 200000)]),
                  dtype=rng.choice(["fp32", "fp32", "bf16"]), drafted=rng.random() < 0.75, ragged=rng.random() < 0.5)
        while work(c)["bytes"] * (c["K"] + 1) > 2 * MOST_BYTES:
            c["B"] = max(1, c["B"] // 2)
        return c
    c |= dict(nkv=nkv, d=d, S=S, block=rng.choice([b for b in (8, 16, 32, 64) if b <= S]),
              codes=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["bf16", "fp16"]))
    if kind == "attention":
        T = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 2000)])
        if T > 9:
            c["B"] = min(c["B"], 4)
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        c |= dict(L=max(T, _log(rng, 1, 131072)), ragged=rng.random() < 0.6, T=T, nh=nh, window=window,
                  sinks=rng.choice([0, 1, 4, 16]) if window else 0, idle=rng.randint(0, c["B"] // 8))
        # the plain form, which pads the rows and holds all scores, has to fit as well
        while (work(c)["bytes"] > MOST_BYTES or work(c)["flops"] > MOST_FLOPS
               or c["B"] * c["L"] * c["nkv"] * c["d"] * 4 > 3 * MOST_BYTES or c["B"] * c["T"] * c["nh"] * c["L"] > 3e8):
            if c["B"] > 1 and (c["T"] > 9 or c["L"] < 200):
                c["B"], c["idle"] = c["B"] // 2, 0
            else:
                c["L"] = max(c["T"], c["L"] // 2)
                c["T"] = c["T"] if c["T"] < 10 or c["L"] > c["T"] else c["T"] // 2
        return c
    c |= dict(T=max(c["B"], _log(rng, 1, 8000 if kind == "write" else 60000)),
              out=rng.choice([c["dtype"], c["dtype"], "fp32"]))
    while work(c)["bytes"] > MOST_BYTES:
        c["T"] = max(c["B"], c["T"] // 2)
    return c


def _rows(c):
    """(slots a row holds, its new tokens) of every row: of the case alone; -1 slots of an idle row."""
    B = c["B"]
    if c["kind"] == "write":  # rows that begin anywhere in a block
        return [(37 * b) % 200 for b in range(B)], [c["T"] // B + (b < c["T"] % B) for b in range(B)]
    if c["kind"] == "read":
        return [(53 * b) % 300 for b in range(B)], [c["T"] // B + (b < c["T"] % B) for b in range(B)]
    L, T = c["L"], c["T"]
    t = [max(1, T - b % T) if c["ragged"] and T < 10 else T for b in range(B)]
    n = [max(1, int(L * (((b + 1) * 0.6180339887) % 1.0))) if c["ragged"] and b else L for b in range(B)]
    n = [max(0, x - y) if T >= 10 else x for x, y in zip(n, t)]
    for i in range(c["idle"]):
        n[B - 1 - 3 * i if B - 1 - 3 * i > 0 else B - 1] = -1
    return n, t


# ------------------------------------------------------------------ inputs
def _tables(n, d):
    ang = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * (
        1.0 / 500000.0 ** (torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d))[None, :]
    return ang.cos().float(), ang.sin().float()


def _pool(need, S, g):
    """(pages in the pool, table [B, W] int32): pages in random order, -1 where a row has none; the
    last page of the pool is nobody's."""
    need = [max(1, -(-n // S)) for n in need]
    W = max(need)
    ids = torch.randperm(sum(need), generator=g, device=DEV).to(torch.int32)
    per = torch.tensor(need, device=DEV)
    used = torch.arange(W, device=DEV)[None, :] < per[:, None]
    start = torch.cumsum(per, 0) - per
    at = (start[:, None] + torch.arange(W, device=DEV)[None, :]).clamp_(max=len(ids) - 1)
    return len(ids) + 1, torch.where(used, ids[at], torch.full_like(ids[at], -1)).contiguous()


def _cached(P, nkv, S, d, block, codes, g):
    """Pages as normal values of different sizes leave them, and their scales."""
    out, scale = torch.empty((P, nkv, S, d), dtype=CODES[codes], device=DEV), []
    per = max(1, (1 << 26) // (nkv * S * d))
    for i in range(0, P, per):
        n = min(per, P - i)
        x = torch.randn((n, nkv, S // block, block, d), generator=g, device=DEV)
        x *= torch.exp(0.4 * torch.randn((n, nkv, S // block, block, 1), generator=g, device=DEV))
        s = x.abs().amax((-2, -1)) / LARGEST[codes]
        x = (x / s[..., None, None]).clamp_(-LARGEST[codes], LARGEST[codes])
        out[i:i + n] = (x.round_() if codes == "int8" else x).view(n, nkv, S, d).to(CODES[codes])
        scale.append(s)
    return out, torch.cat(scale)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "verify":
        B, K, V = c["B"], c["K"], c["V"]
        # a target that favours a few tokens, and a draft model that resembles it
        logits = torch.randn((B, K + 1, V), generator=g, device=DEV) * 1.5
        top = torch.randint(0, max(1, V // 8), (B, K + 1, 8), generator=g, device=DEV)
        top = (top + torch.arange(8, device=DEV) * (V // 8)).clamp_(max=V - 1)
        logits.scatter_add_(2, top, torch.rand((B, K + 1, 8), generator=g, device=DEV) * 14)
        s = dict(kind="verify", target=torch.softmax(logits, -1).to(dt))
        logits = logits[:, :K] + 0.7 * torch.randn((B, K, V), generator=g, device=DEV)
        draft = torch.softmax(logits, -1).to(dt)
        s["tokens"] = torch.multinomial(draft.float().view(B * K, V), 1, generator=g).view(B, K)
        s["draft"] = draft if c["drafted"] else None
        s["accept"] = torch.rand((B, K), generator=g, device=DEV)
        s["sample"] = torch.rand(B, generator=g, device=DEV)
        counts = [max(0, K - b % (K + 1)) for b in range(B)]
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV) if c["ragged"] else None
        return s
    nkv, d, S, block = c["nkv"], c["d"], c["S"], c["block"]
    n, t = _rows(c)
    total, s = sum(t), dict(kind=c["kind"], longest=max(t), codes=c["codes"], block=block)
    P, s["table"] = _pool([max(x, 0) + y for x, y in zip(n, t)], S, g)
    s["lengths"] = torch.tensor(n, dtype=torch.int32, device=DEV)
    s["offsets"] = torch.tensor([sum(t[:b]) for b in range(c["B"] + 1)], dtype=torch.int32, device=DEV)
    s["k_pages"], s["k_scale"] = _cached(P, nkv, S, d, block, c["codes"], g)
    s["v_pages"], s["v_scale"] = _cached(P, nkv, S, d, block, c["codes"], g)
    s["out"] = DTYPES[c.get("out", c["dtype"])]
    s["tokens"] = total
    if c["kind"] != "read":
        count = s["offsets"][1:] - s["offsets"][:-1]
        row = torch.repeat_interleave(torch.arange(c["B"], device=DEV), count.long(), output_size=total)
        s["positions"] = (s["lengths"][row].clamp(min=0) + 11  # eleven tokens came before the cache's first
                          + torch.arange(total, device=DEV) - s["offsets"][row]).to(torch.int32)
        s["cos"], s["sin"] = _tables(max(n) + max(t) + 12, d)
        s["k"], s["v"] = (torch.randn((total, nkv * d), generator=g, device=DEV).to(dt) for _ in range(2))
        if c["kind"] == "attention":
            s["q"] = torch.randn((total, c["nh"] * d), generator=g, device=DEV).to(dt)
            s["window"], s["sinks"] = c["window"], c["sinks"]
    return s


# ------------------------------------------------------------------ the plain forms
def _two_to(e):
    """2^e in 64 bits, of integers within its normal range: exactly."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _on_grid(y, codes):
    """``y`` (64 bits) rounded to the nearest values that a code stands for, ties to even."""
    if codes == "int8":
        return y.round().clamp(-127, 127)
    e = (torch.frexp(y)[1] - 1).clamp(min=-6)
    return ((y * _two_to(3 - e)).round() * _two_to(e - 3)).clamp(-448, 448)


def _rotated(x, cos, sin):
    d2 = x.shape[-1] // 2
    a, b = x[..., :d2], x[..., d2:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _write(s):
    """Every block that gets new tokens, as [rows, blocks, block, kv_heads, d]; those that a row has fewer of go to
    the page that is nobody's."""
    nkv, S, d = s["k_pages"].shape[1:]
    block, codes, most = s["block"], s["codes"], LARGEST[s["codes"]]
    have, first = s["lengths"].long(), s["offsets"][:-1].long()
    new = s["offsets"][1:].long() - first
    nb = (s["longest"] + 2 * block - 2) // block
    slot = ((have.clamp(min=0) // block)[:, None, None] + torch.arange(nb, device=DEV)[:, None]) * block
    slot = slot + torch.arange(block, device=DEV)
    at = slot - have[:, None, None]
    is_new = (at >= 0) & (at < new[:, None, None]) & (have >= 0)[:, None, None]
    fresh = at[:, :, 0] >= 0
    touched = is_new.any(-1)
    page = s["table"].gather(1, (slot[:, :, 0] // S).clamp(max=s["table"].shape[1] - 1)).long()
    page = torch.where(touched, page, len(s["k_pages"]) - 1)
    place = slot[:, :, 0] % S // block
    token = (first[:, None, None] + at).clamp(0, s["tokens"] - 1)
    pos = s["positions"].long()
    key = _rotated(s["k"].view(-1, nkv, d).double(), s["cos"].double()[pos][:, None], s["sin"].double()[pos][:, None])
    for x, pages, scales in ((key, s["k_pages"], s["k_scale"]),
                             (s["v"].view(-1, nkv, d).double(), s["v_pages"], s["v_scale"])):
        x = torch.where(is_new[..., None, None], x[token], 0.0)
        a = x.abs().amax((2, 4))                                                     # [rows, blocks, kv_heads]
        old = torch.where(fresh[..., None], 0.0, scales[page, :, place].double())
        m, e = torch.frexp(a / (most * old))
        grow = torch.where((old > 0) & (a > 0), e - (m == 0.5).to(e.dtype), 0).clamp(min=0)
        begin = torch.where(a > 0, (a / torch.full_like(a, most)).float().clamp(min=SMALLEST_SCALE).double(), 0.0)
        scale = torch.where(old > 0, old * _two_to(grow), begin)
        by_block = pages.view(torch.int8).view(-1, nkv, S // block, block, d)
        there = by_block[page, :, place].view(pages.dtype).transpose(2, 3).double()  # [rows, blocks, block, heads, d]
        there = _on_grid(there * _two_to(-grow)[:, :, None, :, None], codes)
        y = _on_grid(x / torch.where(scale > 0, scale, 1.0)[:, :, None, :, None], codes)
        y = torch.where(is_new[..., None, None], y, there).transpose(2, 3).float().to(pages.dtype)
        by_block[page, :, place] = y.view(torch.int8)
        scales[page, :, place] = scale.float()


def _gathered(s, pages, scales, page, slot):
    """Values [.., kv_heads, d] in 32 bits of slots of pages."""
    x = pages.view(torch.int8)[page, :, slot].view(pages.dtype).float()
    return x * scales[page, :, slot // s["block"]][..., None]


def _read(s):
    S = s["k_pages"].shape[2]
    i = torch.arange(s["tokens"], device=DEV)
    row = torch.searchsorted(s["offsets"][1:].contiguous(), i, right=True)
    slot = s["lengths"][row].long() + i - s["offsets"][row]
    page = s["table"][row, slot // S].long()
    return {n: _gathered(s, s[n + "_pages"], s[n + "_scale"], page, slot % S).flatten(1).to(s["out"]) for n in "kv"}


def _attend(s):
    nkv, S, d = s["k_pages"].shape[1:]
    B, W = s["table"].shape
    T, g = s["longest"], s["q"].shape[1] // (nkv * d)
    have, first = s["lengths"].long(), s["offsets"][:-1].long()
    new = s["offsets"][1:].long() - first
    local = torch.arange(T, device=DEV)
    token = (first[:, None] + local).clamp(max=s["tokens"] - 1)                      # [B, T]
    pos = s["positions"].long()[token]
    q = _rotated(s["q"].view(-1, nkv, g, d).float()[token], s["cos"][pos][:, :, None, None],
                 s["sin"][pos][:, :, None, None])
    q = q.permute(0, 2, 3, 1, 4).reshape(B, nkv, g * T, d) / math.sqrt(d)
    page, slot = s["table"].clamp(min=0).long().repeat_interleave(S, 1), torch.arange(W * S, device=DEV)
    k, v = (_gathered(s, s[n + "_pages"], s[n + "_scale"], page, (slot % S).expand(B, -1)) for n in "kv")
    me = have[:, None] + local
    seen = slot <= me[:, :, None]
    if s["window"]:
        seen = seen & ((slot > me[:, :, None] - s["window"]) | (slot < s["sinks"]))
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(B, nkv, g, T, W * S)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    weight = (score / score.sum(-1, keepdim=True).clamp(min=1e-30)).view(B, nkv, g * T, W * S)
    o = torch.matmul(weight, v.transpose(1, 2).contiguous()).view(B, nkv, g, T, d)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, nkv * g * d)
    row = torch.searchsorted(s["offsets"][1:].contiguous(), torch.arange(s["tokens"], device=DEV), right=True)
    o = o[row, torch.arange(s["tokens"], device=DEV) - first[row]]
    return torch.where((have >= 0)[row, None], o, 0.0).to(s["out"])


def _verify(s):
    p, x = s["target"], s["tokens"]
    B, K, V = p.shape[0], x.shape[1], p.shape[2]
    px = p[:, :K].gather(2, x[:, :, None])[:, :, 0].double()
    qx = 1.0 if s["draft"] is None else s["draft"].gather(2, x[:, :, None])[:, :, 0].double()
    n = torch.full((B,), K, device=DEV) if s["counts"] is None else s["counts"].long()
    good = (s["accept"].double() * qx < px) & (torch.arange(K, device=DEV) < n[:, None])
    accepted = good.long().cumprod(1).sum(1)
    row = torch.arange(B, device=DEV)
    w = p[row, accepted].double()
    refused = accepted < n
    at = accepted.clamp(max=K - 1)
    if s["draft"] is None:
        minus = torch.zeros_like(w).scatter_(1, x[row, at][:, None], 1.0)
    else:
        minus = s["draft"][row, at].double()
    rest = (w - torch.where(refused[:, None], minus, 0.0)).clamp(min=0)
    w = torch.where((rest.amax(1) > 0)[:, None], rest, w)
    upto = w.cumsum(1)
    token = (upto <= (s["sample"].double() * upto[:, -1])[:, None]).sum(1)
    return {"accepted": accepted, "token": token}


def run(state):
    s = state
    if not own:
        if s["kind"] == "verify":
            return _verify(s)
        if s["kind"] == "read":
            return _read(s)
        _write(s)
        return _read(s) if s["kind"] == "write" else _state_of(s, _attend(s))
    if "itmo-final-project_amd" not in sys.path:  # (the working folder is the repository's root)
        sys.path.insert(0, "itmo-final-project_amd")
    import int4_hip

    if s["kind"] == "verify":
        r = int4_hip.verify_drafts(s["target"], s["draft"], s["tokens"], s["accept"], s["sample"], s["counts"])
        return {"accepted": r.accepted, "token": r.token}
    cache = s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["table"]
    if s["kind"] == "attention":
        return _state_of(s, int4_hip.paged_attention8(
            s["q"], s["k"], s["v"], s["cos"], s["sin"], *cache, s["lengths"], s["offsets"], s["positions"],
            longest=s["longest"], window=s["window"] or None, sinks=s["sinks"]))
    if s["kind"] == "write":
        int4_hip.paged_append8(s["k"], s["v"], s["cos"], s["sin"], *cache, s["lengths"], s["offsets"], s["positions"])
    k, v = int4_hip.paged_read8(*cache, s["lengths"], s["offsets"], s["tokens"], s["out"])
    return {"k": k, "v": v}


def _state_of(s, out):
    """An attention's output and the cache that it wrote to: values in units of their blocks' scales, and the scales."""
    r = {n: s[n][:-1] for n in ("k_pages", "v_pages", "k_scale", "v_scale")}  # (the last page is nobody's)
    return {"out": out, **r}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "verify":  # a row of each: that of the first refused draft
        return {"bytes": c["B"] * c["V"] * SIZE[c["dtype"]] * (2 if c["drafted"] else 1), "flops": 4 * c["B"] * c["V"]}
    n, t = _rows(c)
    nkv, d, size = c["nkv"], c["d"], SIZE[c["dtype"]]
    token = 2 * nkv * (d + 4 / c["block"])  # codes and scales of a token
    if c["kind"] == "read":
        return {"bytes": c["T"] * (token + 2 * nkv * d * SIZE[c["out"]]), "flops": 2 * c["T"] * nkv * d}
    if c["kind"] == "write":
        return {"bytes": c["T"] * (2 * token + 2 * nkv * d * (size + SIZE[c["out"]])), "flops": 12 * c["T"] * nkv * d}
    w = c["window"] or 1 << 40

    def seen(i):  # by the token of slot i
        return min(i + 1, w) + max(0, min(c["sinks"], i + 1 - w))

    live = [(x, y) for x, y in zip(n, t) if x >= 0]
    pairs = sum(seen(i) for x, y in live for i in range(x, x + y))
    read = sum(min(x + y, w + y - 1 + c["sinks"]) for x, y in live)
    new = sum(y for _, y in live)
    return {"bytes": read * token + new * (token + 2 * size * (nkv + c["nh"]) * d), "flops": 4 * c["nh"] * d * pairs}


# ------------------------------------------------------------------ in 64 bits
def _steps(x, s, codes):
    """The multiples of the scale ``s`` that stand for ``x``, in 64 bits."""
    y = x / torch.full_like(x, s) if s > 0 else torch.zeros_like(x)  # (not times 1 / s: ties have to stay ties)
    if codes == "int8":
        return torch.clamp(torch.round(y), -127, 127)
    size = y.abs().clamp(min=2.0 ** -6)
    step = size / torch.frexp(size)[0] / 16  # (a power of two by its mantissa: exact, both)
    return torch.clamp(torch.round(y / step) * step, -448, 448)


def _row_values(s, b, n, x):
    """All of row b's ``n`` ("k" or "v"), its new tokens ``x`` [new, kv_heads, d] among them: [slots, kv_heads, d]."""
    S, block, most = s["k_pages"].shape[2], s["block"], LARGEST[s["codes"]]
    have, m = int(s["lengths"][b]), len(x)
    pages = s["table"][b, :-(-(have + m) // S)].long()
    codes = s[n + "_pages"][pages].double().transpose(1, 2).flatten(0, 1)           # [slots, kv_heads, d]
    scale = s[n + "_scale"][pages].double().transpose(1, 2).flatten(0, 1)           # [blocks, kv_heads]
    out = codes * scale.repeat_interleave(block, 0)[:, :, None]
    for j in range(have // block, -(-(have + m) // block)) if m else ():
        lo, hi = max(j * block, have), min((j + 1) * block, have + m)
        for h in range(x.shape[1]):
            mine = x[lo - have:hi - have, h]
            a = float(mine.abs().max())
            if lo == j * block or float(scale[j, h]) == 0.0:
                sc = max(float(torch.tensor(a / most, dtype=torch.float64).float()), SMALLEST_SCALE) if a > 0 else 0.0
            else:
                sc = float(scale[j, h])
                while a > most * sc:
                    sc *= 2.0
                if sc > float(scale[j, h]):
                    past = out[j * block:lo, h]
                    out[j * block:lo, h] = _steps(past, sc, s["codes"]) * sc
            out[lo:hi, h] = _steps(mine, sc, s["codes"]) * sc
    return out[:have + m]


def _fresh(s, b, n):
    """Row b's new keys, rotated, or values: [new, kv_heads, d]."""
    nkv, d = s["k_pages"].shape[1], s["k_pages"].shape[3]
    lo, hi = int(s["offsets"][b]), int(s["offsets"][b + 1])
    x = s[n][lo:hi].double().view(-1, nkv, d)
    return x if n == "v" else _turned(s, x, lo, hi)


def _turned(s, x, lo, hi):
    at = s["positions"][lo:hi].long()
    c, z = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
    x = torch.view_as_complex(torch.stack(x.chunk(2, -1), -1)) * torch.complex(c, z)
    return torch.cat((x.real, x.imag), -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "verify":
        return None  # whole numbers
    nkv, d = c["nkv"], c["d"]
    n, t = _rows(c)
    if c["kind"] == "write" and c["T"] / c["block"] * nkv > 20000:
        return None  # a loop over the blocks takes too long
    if c["kind"] in ("read", "write"):
        got = {"k": [], "v": []}
        for b in range(c["B"]):
            for name in "kv":
                if c["kind"] == "write":
                    got[name].append(_row_values(s, b, name, _fresh(s, b, name))[n[b]:])
                else:
                    empty = torch.empty((0, nkv, d), dtype=torch.float64, device=DEV)
                    s["lengths"][b] = n[b] + t[b]
                    got[name].append(_row_values(s, b, name, empty)[n[b]:])
        return {name: torch.cat(x).flatten(1) for name, x in got.items()}
    out = torch.zeros((sum(t), c["nh"] * d), dtype=torch.float64, device=DEV)
    at = 0
    for b in range(c["B"]):
        lo, at = at, at + t[b]
        if n[b] < 0:
            continue
        k, v = (_row_values(s, b, name, _fresh(s, b, name)) for name in "kv")
        q = _turned(s, s["q"][lo:at].double().view(-1, c["nh"], d), lo, at)
        i = torch.arange(n[b], n[b] + t[b], device=DEV)[:, None]
        j = torch.arange(n[b] + t[b], device=DEV)[None, :]
        hidden = j > i
        if c["window"]:
            hidden = hidden | ((j <= i - c["window"]) & (j >= c["sinks"]))
        for h in range(c["nh"]):
            kv = h // (c["nh"] // nkv)
            p = torch.softmax((q[:, h] @ k[:, kv].T.contiguous() / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
            out[lo:at, h * d:(h + 1) * d] = p @ v[:, kv].contiguous()
    return {"out": out, "k_pages": None, "v_pages": None, "k_scale": None, "v_scale": None}
