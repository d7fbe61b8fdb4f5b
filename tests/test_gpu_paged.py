"""GPU: the operators of the paged key-value cache (int4_hip/paged.py) against a
64-bit statement of them on the CPU."""
import math

import pytest
import torch

import _paged_ref as R
import int4_hip
from _synth import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
# one rounding to the output dtype (as in test_gpu_llama_ops.py)
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# what a probability may be off, relatively: an fp32 score is a sum of d <= 128 products
# (2^-24 each way per addition, |q||k| / sqrt(d) below 40 on these inputs: under 1e-5),
# a probability entering the product with the values in two 16-bit parts 2^-17 (8e-6)
PROB = 2e-5
BOTH = [torch.bfloat16, torch.float16]


def _to(c):
    return {k: None if t is None else t.to(DEV) for k, t in c.items()}


def _same(got, want):
    """Equal values, NaN for NaN."""
    return torch.equal(torch.nan_to_num(got.cpu().float(), nan=7.125, posinf=9e9, neginf=-9e9),
                       torch.nan_to_num(want.float(), nan=7.125, posinf=9e9, neginf=-9e9))


def _check(got, want, mass, dtype, prob=PROB):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and torch.equal(got.isinf(), inf)
    fine = want.isfinite()
    over = (got - want).abs()[fine] - (ROUND[dtype] * want.abs() + prob * mass)[fine] - 1e-7
    assert not over.numel() or over.max().item() <= 0, over.max().item()


def _run(c, dtype, prob=PROB):
    """One call on the GPU against the reference; its tensors, updated by both."""
    g = _to(c)
    out = int4_hip.paged_attention(**g)
    want, mass, _, grown = R.attention(**c)
    assert _same(g["k_pages"], c["k_pages"]) and _same(g["v_pages"], c["v_pages"])
    _check(out, want, mass, dtype, prob)
    if grown is not None:
        got = g["weight"].double().cpu()
        assert torch.equal(got.isnan(), grown.isnan())
        ok = grown.isfinite()
        tol = PROB * c["q"].shape[1] / (c["k"].shape[1]) + 2.0 ** -23 * grown.abs()
        assert ((got - grown).abs()[ok] <= tol[ok]).all()
    return g, out


CASES = [
    # (lengths, heads, kv heads, head_dim, page size): one token and the edges of pages,
    # of eight, of a wave's and of a workgroup's slots; idle rows; one to many query
    # heads per key head; lengths that several workgroups share
    ([0], 1, 1, 64, 8),
    ([-1], 4, 2, 64, 16),
    ([0, 1, -1, 7, 8, 9], 8, 2, 64, 8),
    ([15, 16, 17, 31, 32, 33], 8, 2, 128, 16),
    ([62, 63, 64, 65, -5, 127, 128], 4, 4, 64, 64),
    ([255, 256, 257, 300], 6, 1, 128, 32),
    ([575, 3], 32, 8, 64, 64),
    ([511, 513, 1], 20, 2, 128, 256),
    ([700, 40], 24, 1, 64, 128),
    ([129, 1000], 33, 1, 128, 64),
    ([4097], 8, 2, 64, 64),
    ([5000, 2, 2500], 12, 4, 128, 1024),
    ([9001], 2, 1, 128, 16),
]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lens,nh,nkv,d,S", CASES)
def test_attention(dtype, lens, nh, nkv, d, S):
    print(f"[paged attention] {dtype} {lens} {nh}/{nkv}x{d} S={S}", flush=True)
    for weights in (True, False):
        _run(R.attention_case(lens, nh, nkv, d, S, dtype, seed=len(lens) + nh, weights=weights), dtype)


@pytest.mark.parametrize("dtype", BOTH)
def test_attention_many_rows(dtype):
    lens = [(37 * i) % 211 - 1 for i in range(150)]
    print(f"[paged attention] {dtype} 150 rows", flush=True)
    _run(R.attention_case(lens, 4, 2, 64, 16, dtype, seed=1), dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("nh,nkv,d", [(8, 4, 64), (16, 4, 128), (36, 4, 64)])
def test_attention_more_rows_than_the_chip_holds(dtype, nh, nkv, d):
    """Workgroups of one wave; two rows long enough that several share them, one of them with a page outside the pool."""
    lens = [(13 * i) % 71 - 1 for i in range(140)]
    lens[3], lens[70], lens[139] = 1500, 129, 4000 * 64 // d
    print(f"[paged attention] {dtype} 140 rows of {nh}/{nkv}x{d}", flush=True)
    for weights in (True, False):
        c = R.attention_case(lens, nh, nkv, d, 32, dtype, seed=nh, weights=weights)
        c["table"][139, 17] = c["k_pages"].shape[0]
        c["v_pages"][c["table"][3, 30], 1, 3, 5] = math.inf
        out = int4_hip.paged_attention(**_to(c))
        want, mass, reach, _ = R.attention(**c)
        rest = torch.arange(140) != 3
        _check(out.cpu()[rest], want[rest], mass[rest], dtype)
        # beside an infinity as in test_attention_not_finite
        prob = (2.0 ** -8 * (1 + reach[3].clamp(max=40).max())).item()
        _check(out[3], want[3], mass[3].nan_to_num(0, 0, 0), dtype, prob)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lens,nh,nkv", [([0, 5, -1, 64], 17, 1), ([3000, 129, 1], 32, 1), ([5000, 255], 33, 1),
                                         ([700, 9000], 80, 2), ([20, 66] * 40 + [2000], 100, 5),
                                         ([20, 66] * 60 + [2000], 100, 5)])
def test_attention_many_query_heads_a_key_head(dtype, lens, nh, nkv):
    print(f"[paged attention] {dtype} {len(lens)} rows of {nh}/{nkv}x64", flush=True)
    for weights in (True, False):
        c = R.attention_case(lens, nh, nkv, 64, 64, dtype, seed=nh, weights=weights)
        if len(lens) == 4:
            c["table"][3, 0] = -1
        _run(c, dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("B,nh,nkv,d,S,width", [(5, 8, 2, 64, 64, 4), (5, 8, 2, 64, 64, 5), (5, 8, 1, 128, 32, 4),
                                                (5, 8, 1, 128, 128, 1), (5, 24, 1, 64, 8, 3), (5, 24, 1, 128, 64, 2),
                                                (150, 4, 4, 64, 16, 16), (150, 8, 4, 128, 8, 16)])
def test_attention_weights_of_narrow_tables(dtype, B, nh, nkv, d, S, width):
    """Rows up to the last slot of tables that one workgroup has whole, and of tables just wider."""
    cap = width * S
    lens = [[cap - 1, 0, -1, cap // 2, 3, cap - 2, 7][i % 7] for i in range(B)]
    print(f"[paged attention] {dtype} {B} rows of {width}x{S}, {nh}/{nkv}x{d}", flush=True)
    c = R.attention_case(lens, nh, nkv, d, S, dtype, seed=B + width, weights=True, width=width)
    c["table"] = c["table"][:, :width].contiguous()
    c["table"][3, 0] = -1
    c["positions"][4] = len(c["cos"])
    _run(c, dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("B,nh,nkv,S,width", [(6, 17, 1, 64, 4), (6, 33, 1, 64, 4), (150, 100, 5, 16, 16),
                                              (150, 132, 4, 32, 2), (600, 24, 1, 8, 9), (9, 64, 2, 256, 1)])
def test_attention_weights_of_narrow_tables_and_wide_groups(dtype, B, nh, nkv, S, width):
    test_attention_weights_of_narrow_tables(dtype, B, nh, nkv, 64, S, width)


@pytest.mark.parametrize("dtype", BOTH)
def test_attention_steps_accumulate(dtype):
    """Several steps, lengths growing across a page's end: every step's state feeds the next."""
    lens = [14, 0, 30]
    c = R.attention_case(lens, 8, 2, 64, 16, dtype, seed=3, width=4, spare=8)
    # pages for the growth
    used = set(c["table"][c["table"] >= 0].tolist())
    free = [p for p in range(c["k_pages"].shape[0]) if p not in used]
    for b in range(3):
        for i in range(c["table"].shape[1]):
            if c["table"][b, i] < 0 and free:
                c["table"][b, i] = free.pop()
    for step in range(4):
        c["q"], c["k"], c["v"] = (randn(c[x].shape, 100 * step + i, dtype=dtype) for i, x in enumerate("qkv"))
        g, _ = _run(c, dtype)
        c["weight"] = g["weight"].cpu()
        c["lengths"] = c["lengths"] + 1
        c["positions"] = c["positions"] + 1


@pytest.mark.parametrize("dtype", BOTH)
def test_attention_strided_projections(dtype):
    """q, k, v as slices of one projection, and as operands that need a copy."""
    c = R.attention_case([40, 5], 8, 2, 64, 16, dtype, seed=5)
    ref = int4_hip.paged_attention(**_to(c))
    g = _to(c)
    fused = torch.cat([g["q"], g["k"], g["v"]], 1)
    n, m = c["q"].shape[1], c["k"].shape[1]
    out = int4_hip.paged_attention(**dict(g, q=fused[:, :n], k=fused[:, n:n + m], v=fused[:, n + m:]))
    assert torch.equal(out, ref)
    g = _to(c)
    odd = torch.zeros((2, n + 3), dtype=dtype, device=DEV)
    odd[:, 1:n + 1] = g["q"]
    wide = torch.zeros((2, 2 * m), dtype=dtype, device=DEV)
    wide[:, ::2] = g["v"]
    out = int4_hip.paged_attention(**dict(g, q=odd[:, 1:n + 1], v=wide[:, ::2],
                                          k=g["k"].t().contiguous().t()))
    assert torch.equal(out, ref)
    one = _to(R.attention_case([40, 5], 8, 2, 64, 16, dtype, seed=5))
    out = int4_hip.paged_attention(**dict(one, q=g["q"][:1].expand(2, n)))  # a broadcast query
    want = R.attention(**dict(R.attention_case([40, 5], 8, 2, 64, 16, dtype, seed=5), q=c["q"][:1].expand(2, n)))
    _check(out, want[0], want[1], dtype)


def test_attention_shared_prefix():
    """Two rows that read the same pages, each with a page of its own behind them."""
    dtype = torch.bfloat16
    c = R.attention_case([32, 40], 8, 2, 64, 16, dtype, seed=6, weights=False)
    c["table"][1, :2] = c["table"][0, :2]
    _run(c, dtype)


@pytest.mark.parametrize("dtype", BOTH)
def test_attention_out_of_range(dtype):
    """A slot past the table, positions outside the tables, pages outside the pool: NaN rows,
    the others as ever, and nothing written for a refused token."""
    lens = [20, 32, 5, 5, 40, 40, 9]
    c = R.attention_case(lens, 4, 2, 64, 16, dtype, seed=7, width=3)
    c["table"] = c["table"][:, :3].contiguous()
    c["lengths"][1] = 48                          # slot 48 of a table of 3 x 16
    c["positions"][2], c["positions"][3] = -1, len(c["cos"])
    c["table"][4, 0] = c["k_pages"].shape[0]      # an old page
    c["table"][5, 2] = -3                         # the new token's page
    before = c["weight"].clone()
    g, out = _run(c, dtype)
    assert out[[1, 2, 3, 4, 5]].isnan().all() and not out[[0, 6]].isnan().any()
    for b in (4, 5):
        for i in range(3):
            p = int(c["table"][b, i])
            if 0 <= p < len(before) and not (b == 4 and i == 2):
                assert _same(g["weight"][p], before[p])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("where", ["value", "key", "query", "new value"])
def test_attention_not_finite(dtype, where):
    """Infinities and NaN among what is attended to come through as in the formula."""
    c = R.attention_case([50, 50, 700, 50], 8, 2, 64, 16, dtype, seed=8)
    for b, bad in enumerate((math.inf, -math.inf, math.inf, math.nan)):
        if where == "query":
            c["q"][b, 7] = bad
        elif where == "new value":
            c["v"][b, 3] = bad
        else:
            p, s = int(c["table"][b, 1]), 5
            (c["v_pages"] if where == "value" else c["k_pages"])[p, 1, s, 9] = bad
    g = _to(c)
    out = int4_hip.paged_attention(**g)
    want, mass, reach, grown = R.attention(**c)
    # beside an infinity the operands may enter in one 16-bit part: 2^-8 of a score's terms
    prob = (2.0 ** -8 * (1 + reach.nan_to_num(0, 0, 0).clamp(max=40).max())).item()
    _check(out, want, mass.nan_to_num(0, 0, 0), dtype, prob)
    got = g["weight"].cpu()
    assert torch.equal(got.isnan(), grown.isnan())


def test_attention_infinite_key_scores_minus_infinity():
    """A key whose score is -inf weighs nothing, alone among finite ones, and where all are: NaN."""
    dtype = torch.bfloat16
    c = R.attention_case([30], 2, 1, 64, 16, dtype, seed=9)
    c["positions"][:] = 0  # no rotation
    c["q"][:] = c["q"].abs() + 0.25
    c["k_pages"][int(c["table"][0, 0]), 0, 3] = -math.inf
    g = _to(c)
    out = int4_hip.paged_attention(**g)
    want, mass, _, grown = R.attention(**c)
    assert want.isfinite().all()
    _check(out, want, mass, dtype, 2.0 ** -3)
    assert g["weight"][int(c["table"][0, 0]), 0, 3].item() == grown[int(c["table"][0, 0]), 0, 3].item()
    c["k"][:] = -math.inf
    for i in range(2):
        c["k_pages"][int(c["table"][0, i])] = -math.inf
    assert int4_hip.paged_attention(**_to(c)).isnan().all()


def test_attention_large_scores():
    """Scores far apart, the largest first and last: the running maximum is carried."""
    dtype = torch.float16
    for first in (True, False):
        c = R.attention_case([600], 4, 1, 64, 64, dtype, seed=10)
        big = c["k_pages"][int(c["table"][0, 0 if first else 9])]
        big[0, 0 if first else 20] *= 30
        _run(c, dtype, prob=30 * PROB)


def test_attention_repeats_bit_for_bit():
    c = R.attention_case([9000, 100, 3000], 32, 8, 64, 64, torch.bfloat16, seed=11)
    g = _to(c)
    w = g["weight"].clone()
    first = int4_hip.paged_attention(**g)
    w1 = g["weight"].clone()
    for _ in range(5):
        g["weight"].copy_(w)
        assert torch.equal(int4_hip.paged_attention(**g), first)
        assert _same(g["weight"], w1.cpu())


def test_attention_offsets_past_32_bits():
    """Pages whose bytes and elements lie beyond 2^32, in a pool mostly untouched."""
    dtype = torch.bfloat16
    c = R.attention_case([200, 33], 8, 2, 64, 64, dtype, seed=12)
    P = c["k_pages"].shape[0]
    many = (1 << 32) // (2 * 64 * 64) + 5 * P
    shift = many - P
    g = _to(c)
    for name in ("k_pages", "v_pages", "weight"):
        big = torch.empty((many, *g[name].shape[1:]), dtype=g[name].dtype, device=DEV)
        big[shift:] = g[name]
        g[name] = big
    g["table"] = torch.where(g["table"] >= 0, g["table"] + shift, g["table"])
    out = int4_hip.paged_attention(**g)
    n = int4_hip.paged_evict(g["k_pages"], g["v_pages"], g["weight"], g["table"], g["lengths"],
                             torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV), 100, 10)
    want, mass, _, _ = R.attention(**c)
    _check(out, want, mass, dtype)
    assert _same(g["k_pages"][shift:], c["k_pages"]) and n.tolist() == [100, 33]
    c["weight"] = g["weight"][shift:].cpu()
    new = torch.tensor([[P, P + 1], [P + 2, P + 3]], dtype=torch.int32)
    more = [torch.cat([t, torch.zeros((4, *t.shape[1:]), dtype=t.dtype)]) for t in
            (c["k_pages"], c["v_pages"], c["weight"])]
    R.evict(*more, c["table"], c["lengths"], new, 100, 10)
    for i, name in enumerate(("k_pages", "v_pages", "weight")):
        assert _same(g[name][2, :, :33], more[i][P + 2, :, :33]) and _same(g[name][0], more[i][P])


def test_attention_on_another_stream_and_in_a_graph():
    c = R.attention_case([70, 5, 300], 8, 2, 128, 16, torch.bfloat16, seed=13)
    want = int4_hip.paged_attention(**_to(c))
    g = _to(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = int4_hip.paged_attention(**g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    g = _to(c)
    start = g["weight"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = int4_hip.paged_attention(**g)
    weights = None
    for i in range(4):
        g["weight"].copy_(start)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert weights is None or _same(g["weight"], weights)
        weights = g["weight"].cpu()
        int4_hip.paged_attention(**_to(c))  # the program's own work between replays
    # other lengths, same graph
    c2 = R.attention_case([70, 5, 300], 8, 2, 128, 16, torch.bfloat16, seed=13)
    c2["lengths"] = torch.tensor([12, -1, 299], dtype=torch.int32)
    g["lengths"].copy_(c2["lengths"])
    graph.replay()
    c2w, mass, _, _ = R.attention(**dict(c2, weight=None))
    _check(out, c2w, mass, torch.bfloat16)


def test_empty_batch():
    c = _to(R.attention_case([3], 4, 2, 64, 16, torch.bfloat16, seed=14))
    for k in ("q", "k", "v", "table", "lengths", "positions"):
        c[k] = c[k][:0]
    assert int4_hip.paged_attention(**c).shape == (0, 256)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    int4_hip.paged_append(c["k"], c["v"], c["cos"], c["sin"], c["k_pages"], c["v_pages"], c["table"], none, none, none)
    assert int4_hip.paged_evict(c["k_pages"], c["v_pages"], c["weight"], c["table"], none, c["table"], 4, 2).shape == (0,)


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("T,nkv,d,S", [(1, 1, 64, 8), (13, 2, 128, 16), (100, 3, 64, 64), (1000, 8, 128, 32),
                                       (777, 1, 64, 1024)])
def test_append(dtype, T, nkv, d, S):
    print(f"[paged append] {dtype} T={T} {nkv}x{d} S={S}", flush=True)
    lens = [T // 2 + 5, T - T // 2 + 3]
    P, table = R.pages_for(lens, S, T)
    kp, vp = (randn((P, nkv, S, d), i, dtype=dtype) for i in (1, 2))
    w = randn((P, nkv, S), 3, dtype=torch.float32)
    cos, sin = R.tables(T + 50, d)
    k, v = (randn((T, nkv * d), i, dtype=dtype) for i in (4, 5))
    rows = (torch.arange(T) % 2).int()
    slots = (torch.arange(T) // 2 + 3).int()
    positions = slots + 31
    perm = torch.randperm(T, generator=torch.Generator().manual_seed(T))
    k, v, rows, slots, positions = k[perm], v[perm], rows[perm].contiguous(), slots[perm], positions[perm]
    skip = []
    if T >= 13:  # padding and what is out of range is left out
        rows[2], slots[3], positions[4], rows[5] = -1, -9, -1, 2
        slots[6], positions[7] = table.shape[1] * S, len(cos)
        skip = [2, 3, 4, 5, 6, 7]
    for weight in (w, None):
        g = [t.to(DEV) for t in (kp, vp)]
        gw = None if weight is None else weight.to(DEV)
        int4_hip.paged_append(k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), *g, table.to(DEV), rows.to(DEV),
                              slots.to(DEV), positions.to(DEV), weight=gw)
        wk, wv, ww = kp.clone(), vp.clone(), w.clone()
        for t in range(T):
            if t in skip:
                continue
            p, s = int(table[int(rows[t]), int(slots[t]) // S]), int(slots[t]) % S
            wk[p, :, s] = R.rope32(k[t].float().view(nkv, d), cos[positions[t]], sin[positions[t]]).to(dtype)
            wv[p, :, s] = v[t].view(nkv, d)
            ww[p, :, s] = 0.0
        assert torch.equal(g[0].cpu(), wk) and torch.equal(g[1].cpu(), wv)
        assert gw is None or torch.equal(gw.cpu(), ww)


def test_append_skips_pages_outside_the_pool_and_takes_strided_rows():
    dtype, nkv, d, S = torch.bfloat16, 2, 64, 16
    table = torch.tensor([[0, 9, -1, 2]], dtype=torch.int32, device=DEV)
    kp, vp = (torch.zeros((3, nkv, S, d), dtype=dtype, device=DEV) for _ in range(2))
    cos, sin = (t.to(DEV) for t in R.tables(64, d))
    fused = randn((64, 3 * nkv * d), 1, dtype=dtype).to(DEV)
    k, v = fused[:, nkv * d:2 * nkv * d], fused[:, 2 * nkv * d:]
    i = torch.arange(64, dtype=torch.int32, device=DEV)
    int4_hip.paged_append(k, v, cos, sin, kp, vp, table, torch.zeros_like(i), i, torch.zeros_like(i))
    assert torch.equal(kp[0], k[:16].view(16, nkv, d).transpose(0, 1)) and not kp[1].any()
    assert torch.equal(vp[2], v[48:].view(16, nkv, d).transpose(0, 1))


# ---------------------------------------------------------------- eviction
def _evict(lens, nkv, d, S, keep, recent, dtype, seed, fix=None, width=None):
    B = len(lens)
    P, both = R.pages_for([max(n, 0) for n in lens] + [keep] * B, S, seed, width=width)
    table = both[:B].contiguous()
    new = both[B:, :-(-keep // S)].contiguous()
    kp, vp = (randn((P, nkv, S, d), seed + i, dtype=dtype) for i in (1, 2))
    w = randn((P, nkv, S), seed + 3, dtype=torch.float32).abs()
    if fix:
        fix(w)
    lengths = torch.tensor(lens, dtype=torch.int32)
    g = [t.to(DEV) for t in (kp, vp, w)]
    n = int4_hip.paged_evict(*g, table.to(DEV), lengths.to(DEV), new.to(DEV), keep, recent)
    want = R.evict(kp, vp, w, table, lengths, new, keep, recent)
    assert torch.equal(n.cpu(), want)
    for a, b in zip(g, (kp, vp, w)):
        assert _same(a, b)


@pytest.mark.parametrize("width,S", [(20000, 8), (300, 64), (130, 128), (40, 1024), (513, 64), (2100, 8)])
@pytest.mark.parametrize("lens,nkv,keep,recent", [([1], 1, 1, 0), ([5, 0, -1, 9], 2, 4, 2), ([64, 65, 63], 2, 64, 64),
                                                  ([300, 299, 12, 301], 3, 299, 10), ([1000, 1025, 2048], 2, 77, 0),
                                                  ([2000, 4099], 2, 1025, 1024), ([15000, 8193], 1, 6001, 300)])
def test_evict_from_wide_tables(width, S, lens, nkv, keep, recent):
    """Short rows of tables of every width: what is launched follows the table."""
    print(f"[paged eviction] {lens} of {width}x{S}, keep {keep} / {recent}", flush=True)
    _evict(lens, nkv, 64, S, keep, recent, torch.float16, seed=width, width=width)


@pytest.mark.parametrize("keep,recent,levels", [(40000, 500, 0), (100, 0, 0), (69900, 100, 0), (33000, 0, 7),
                                                (20000, 1000, 1), (30000, 11, 30000)])
def test_evict_rows_longer_than_the_selection_holds(keep, recent, levels):
    """Keys read in several runs; with `levels` the weights are of so many values only."""
    def fix(w):
        if levels:
            w.copy_((w * levels).floor().clamp(max=levels - 1))
    print(f"[paged eviction] 70001, keep {keep} / {recent}, {levels} levels", flush=True)
    _evict([70001, 33000 + recent, 32768 + recent], 2, 64, 256, keep, recent, torch.bfloat16, seed=keep, fix=fix)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lens,nkv,d,S,keep,recent", [
    ([1], 1, 64, 8, 1, 0), ([5, 0, -1, 9], 2, 64, 8, 4, 2), ([64, 65, 63], 2, 128, 16, 64, 64),
    ([300, 299, 12, 301], 3, 64, 32, 299, 10), ([1000], 8, 128, 64, 77, 0), ([2000, 4099], 2, 64, 64, 1025, 1024),
    ([257, 256, 255], 1, 128, 256, 100, 100), ([70], 2, 64, 16, 200, 5), ([20011], 1, 64, 128, 6001, 300)])
def test_evict(dtype, lens, nkv, d, S, keep, recent):
    print(f"[paged evict] {dtype} {lens} {nkv}x{d} S={S} keep={keep} recent={recent}", flush=True)
    _evict(lens, nkv, d, S, keep, recent, dtype, seed=sum(map(abs, lens)))


@pytest.mark.parametrize("name", ["equal", "zeros", "few values", "signs", "nan", "infinite", "close"])
def test_evict_ties_and_odd_weights(name):
    def fix(w):
        if name == "equal":
            w.fill_(0.25)
        elif name == "zeros":
            w[torch.rand(w.shape, generator=torch.Generator().manual_seed(1)) < 0.9] = 0.0
            w[torch.rand(w.shape, generator=torch.Generator().manual_seed(2)) < 0.3] *= -0.0
        elif name == "few values":
            w.copy_((w * 3).floor())
        elif name == "signs":
            w.mul_(torch.where(torch.rand(w.shape, generator=torch.Generator().manual_seed(3)) < 0.5, -1.0, 1.0))
        elif name == "nan":
            w[torch.rand(w.shape, generator=torch.Generator().manual_seed(4)) < 0.2] = math.nan
            w[torch.rand(w.shape, generator=torch.Generator().manual_seed(5)) < 0.1] = -math.nan
        elif name == "infinite":
            w[torch.rand(w.shape, generator=torch.Generator().manual_seed(6)) < 0.2] = math.inf
            w[torch.rand(w.shape, generator=torch.Generator().manual_seed(7)) < 0.2] = -math.inf
        else:  # neighbours in the last bits
            w.copy_((torch.full_like(w, 1.0).view(torch.int32) + (w * 100).int() % 7).view(torch.float32))
    for keep, recent in ((100, 20), (700, 0), (1, 0), (999, 1)):
        _evict([1000, 333, 701], 2, 64, 16, keep, recent, torch.bfloat16, seed=keep, fix=fix)


def test_evict_past_the_table_and_bad_pages():
    dtype = torch.bfloat16
    kp, vp = (randn((8, 1, 16, 64), i, dtype=dtype).to(DEV) for i in (1, 2))
    w = torch.rand((8, 1, 16), device=DEV)
    table = torch.tensor([[0, 1], [2, 99], [3, 0]], dtype=torch.int32, device=DEV)
    new = torch.tensor([[4], [5], [-2]], dtype=torch.int32, device=DEV)
    k0, w0 = kp.clone(), w.clone()
    n = int4_hip.paged_evict(kp, vp, w, table, torch.tensor([33, 30, 20], dtype=torch.int32, device=DEV), new, 16, 4)
    assert n.tolist() == [-1, 16, 16]
    assert torch.equal(kp[:5], k0[:5]) and torch.equal(kp[6:], k0[6:]) and torch.equal(w[:5], w0[:5])
    # of row 1 the slots 26..29 lie outside the pool; the kept ones among 0..15 are copied
    early = sorted(sorted(range(16), key=lambda j: -w0[2, 0, j].item())[:12])
    assert torch.equal(kp[5, 0, :12], k0[2, 0, early]) and torch.equal(kp[5, 0, 12:], k0[5, 0, 12:])


def test_evicted_cache_is_attended_to():
    """Append, attend, evict, attend: the path of a sequence over its budget."""
    dtype, nkv, nh, d, S, n = torch.bfloat16, 2, 8, 64, 16, 100
    P = 24
    kp, vp, w = torch.zeros((P, nkv, S, d), dtype=dtype), torch.zeros((P, nkv, S, d), dtype=dtype), torch.zeros(P, nkv, S)
    table = torch.arange(8, dtype=torch.int32)[None]
    new = torch.arange(8, 16, dtype=torch.int32)[None]
    cos, sin = R.tables(200, d)
    g = _to(dict(kp=kp, vp=vp, w=w, table=table, new=new, cos=cos, sin=sin))
    k, v = (randn((n, nkv * d), i, dtype=dtype).to(DEV) for i in (1, 2))
    i = torch.arange(n, dtype=torch.int32, device=DEV)
    int4_hip.paged_append(k, v, g["cos"], g["sin"], g["kp"], g["vp"], g["table"], torch.zeros_like(i), i, i, weight=g["w"])
    one = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)  # noqa: E731

    def step(tab, length, pos, seed):
        x = [randn((1, m * d), seed + j, dtype=dtype) for j, m in enumerate((nh, nkv, nkv))]
        c = dict(q=x[0], k=x[1], v=x[2], cos=cos, sin=sin, k_pages=g["kp"].cpu(), v_pages=g["vp"].cpu(),
                 table=tab.cpu(), lengths=one(length).cpu(), positions=one(pos).cpu(), weight=g["w"].cpu())
        out = int4_hip.paged_attention(*[t.to(DEV) for t in x], g["cos"], g["sin"], g["kp"], g["vp"], tab, one(length),
                                       one(pos), weight=g["w"])
        want, mass, _, grown = R.attention(**c)
        _check(out, want, mass, dtype)
        assert (g["w"].cpu() - grown).abs().max() < 1e-4

    for t in range(3):
        step(g["table"], n + t, n + t, 10 * t)
    m = int4_hip.paged_evict(g["kp"], g["vp"], g["w"], g["table"], one(n + 3), g["new"], 40, 8)
    assert m.tolist() == [40]
    for t in range(3):
        step(g["new"], 40 + t, n + 3 + t, 100 + 10 * t)


# ---------------------------------------------------------------- refusals
@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 256)), dict(q=torch.zeros(2, 200, dtype=torch.bfloat16)),
    dict(q=torch.zeros(3, 256, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 0, dtype=torch.bfloat16)),
    dict(k=torch.zeros(2, 256, dtype=torch.bfloat16)), dict(lengths=torch.zeros(2, dtype=torch.int64)),
    dict(lengths=torch.zeros(3, dtype=torch.int32)), dict(positions=torch.zeros(2)),
    dict(table=torch.zeros(2, 3, dtype=torch.int64)), dict(table=torch.zeros(2, 0, dtype=torch.int32)),
    dict(cos=torch.zeros(5, 32, dtype=torch.float64)), dict(sin=torch.zeros(5, 16)),
    dict(weight=torch.zeros(2, 2, 16)), dict(k_pages=torch.zeros(4, 2, 16, 64)),
    dict(v_pages=torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)[..., ::2])])
def test_attention_refuses(change):
    c = R.attention_case([5, 2], 4, 2, 64, 16, torch.bfloat16, seed=1)
    int4_hip.paged_attention(**_to(c))
    with pytest.raises(AssertionError):
        int4_hip.paged_attention(**dict(_to(c), **_to(change)))
    with pytest.raises(AssertionError):  # another device
        int4_hip.paged_attention(**dict(_to(c), q=c["q"]))


@pytest.mark.parametrize("S,d", [(24, 64), (4, 64), (2048, 64), (16, 32), (16, 96)])
def test_caches_of_other_forms_are_refused(S, d):
    """By every operator as a caller's mistake, before anything is launched."""
    z = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device=DEV)
    i = z(2, dtype=torch.int32)
    pages, table, w = [z(4, 2, S, d), z(4, 2, S, d)], z(2, 2, dtype=torch.int32), z(4, 2, S, dtype=torch.float32)
    cos = z(9, d // 2, dtype=torch.float32)
    with pytest.raises(AssertionError):
        int4_hip.paged_append(z(2, 2 * d), z(2, 2 * d), cos, cos, *pages, table, i, i, i)
    with pytest.raises(AssertionError):
        int4_hip.paged_attention(z(2, 4 * d), z(2, 2 * d), z(2, 2 * d), cos, cos, *pages, table, i, i, w)
    with pytest.raises(AssertionError):
        int4_hip.paged_evict(*pages, w, table, i, table, 4, 1)


def test_append_and_evict_refuse():
    c = _to(R.attention_case([5, 2], 4, 2, 64, 16, torch.bfloat16, seed=1))
    i = torch.zeros(2, dtype=torch.int32, device=DEV)
    cache = [c[k] for k in ("cos", "sin", "k_pages", "v_pages", "table")]
    for k, v, *idx in ((c["q"], c["v"], i, i, i), (c["k"], c["v"].float(), i, i, i), (c["k"], c["v"], i.long(), i, i),
                       (c["k"], c["v"], i, i[:1], i), (c["k"][:1], c["v"], i, i, i), (c["k"], c["v"], i, i, i.cpu())):
        with pytest.raises(AssertionError):
            int4_hip.paged_append(k, v, *cache, *idx)
    pages = [c["k_pages"], c["v_pages"]]
    for keep, recent in ((0, 0), (4, 5), (4, -1), (10 ** 6, 0)):
        with pytest.raises(AssertionError):
            int4_hip.paged_evict(*pages, c["weight"], c["table"], c["lengths"], c["table"], keep, recent)
    with pytest.raises(AssertionError):
        int4_hip.paged_evict(*pages, None, c["table"], c["lengths"], c["table"], 4, 1)
    with pytest.raises(AssertionError):
        int4_hip.paged_evict(*pages, c["weight"], c["table"], c["lengths"], c["table"][:1], 4, 1)
