"""GPU: the operators of the 8-bit paged cache (int4_hip/paged8.py) against a 64-bit
statement of them on the CPU."""
import pytest
import torch

import _paged8_ref as R
import int4_hip
from _paged8_ref import CODES, MOST, NAN
from _synth import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = [torch.bfloat16, torch.float16]
CACHE = ("k_pages", "v_pages", "k_scale", "v_scale")
IDS = {torch.int8: "int8", torch.float8_e4m3fn: "e4m3", torch.bfloat16: "bf16", torch.float16: "fp16"}


def ids(x):
    return IDS.get(x, str(x))


def _to(c):
    return {k: t.to(DEV) if isinstance(t, torch.Tensor) else t for k, t in c.items()}


def _call(f, c, *names):
    return f(*(c[n] for n in names))


def _append(c):
    int4_hip.paged_append8(*(c[n] for n in ("k", "v", "cos", "sin") + CACHE +
                             ("table", "lengths", "offsets", "positions")))


def _same_cache(got, want):
    """Equal codes (zeros of either sign) and scales, NaN for NaN."""
    for n in CACHE:
        a, b = got[n].cpu().float(), want[n].float()
        assert torch.equal(a.isnan(), b.isnan()), n
        bad = torch.nan_to_num(a) != torch.nan_to_num(b)
        assert not bad.any(), (n, bad.nonzero()[:4], a[bad][:4], b[bad][:4])


def _check(got, want, mass, reach, dtype, slots, d):
    """One rounding to the dtype, eps / 2 = half a step; and the fp32 sums before it.

    A score is a sum of d products of rotated queries (two products and their sum each:
    3 roundings), in 3 d / 32 matrix instructions that round some 32 partial sums each: at most
    (3 + 3 d) 2^-24 reach, times the scale and 1 / sqrt(d): 2 more.  An exponential: 2^-22 and
    what its argument's rounding makes, 2^-24 of it, 2 reach at most.  Probabilities times
    scales enter with 24 bits: 3 roundings; sums over the slots: one a unit of 32 and part.
    All of it twice, in the sum and in the denominator.
    """
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), (got.isnan() != want.isnan()).nonzero()[:5]
    score = (5 + 3 * d + 2) * 2.0 ** -24 * reach
    prob = 2 * (score + 2.0 ** -22 + (16 + 3 * slots / 32) * 2.0 ** -24)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + prob * mass + torch.finfo(dtype).tiny
    # the nearest number of a dtype to what lies half a step past its largest is infinity
    past = got.isinf()
    edge = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)
    assert (torch.sign(got[past]) * want[past] + tol[past] >= edge).all()
    over = ((got - want).abs() - tol)[~want.isnan() & ~past]
    assert not over.numel() or over.max().item() <= 0, over.max().item()


def _run(c, dtype, **more):
    """One call on the GPU against the reference; its tensors, updated by both."""
    g = _to(c)
    out = int4_hip.paged_attention8(**g, **more)
    want, mass, reach = R.attention(**c)
    _same_cache(g, c)
    assert out.dtype == dtype and out.shape == want.shape
    _check(out, want, mass, reach, dtype, c["table"].shape[1] * c["k_pages"].shape[2], c["k_pages"].shape[3])
    return g, out


# ---------------------------------------------------------------- append and read
@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("dtype", BOTH, ids=ids)
@pytest.mark.parametrize("nkv,d,S,block", [(2, 64, 16, 8), (3, 128, 64, 64), (1, 64, 64, 32), (5, 128, 32, 16),
                                           (2, 64, 128, 64), (9, 128, 8, 8)])
def test_append_is_the_definition(kind, dtype, nkv, d, S, block):
    """Prompts that begin anywhere, blocks that are full, begun and continued; every code and scale equal."""
    lens, new = [0, 5, block - 1, block, 2 * block + 3, 0, 7, -1], [1, 2 * block, 1, block + 2, 3, 0, 1, 4]
    c = R.case(lens, new, nkv, nkv, d, S, block, kind, dtype, seed=nkv)
    g = _to(c)
    _append(g)
    R.append(**c)
    _same_cache(g, c)


@pytest.mark.parametrize("kind", CODES, ids=ids)
def test_append_token_by_token_grows_the_scales(kind):
    """Values that grow, shrink, vanish and jump: scales double, codes are rounded again, each step as defined."""
    sizes = [0.0, 1e-3, 1.0, 0.5, 3.0, 2.9, 200.0, 1e-30, 201.0, 6e4, 1e30, 0.0]
    c = R.case([3], [1], 2, 2, 64, 32, 16, kind, torch.bfloat16, seed=4, width=2, angles=64)
    c["table"] = torch.tensor([[2, 0]], dtype=torch.int32)
    g = _to(c)
    for i, size in enumerate(sizes):
        for n in ("k", "v"):
            x = (randn((1, 2 * 64), seed=50 + i) * size).bfloat16()
            c[n], g[n] = x, x.to(DEV)
        c["lengths"] = torch.tensor([3 + i], dtype=torch.int32)
        g["lengths"] = c["lengths"].to(DEV)
        _append(g)
        R.append(**c)
        _same_cache(g, c)


@pytest.mark.parametrize("kind", CODES, ids=ids)
def test_append_of_values_between_two_codes(kind):
    """Values whose quotient by the scale is the middle between two codes exactly: to the even one."""
    most, nkv, d = MOST[kind], 1, 64
    scale = 3.0 * 2.0 ** -4
    steps = [n + 0.5 for n in range(-12, 12)] if kind == torch.int8 else [x * 17 / 16 for x in (1, 2, 4, 8)] + [
        19 / 16, -21 / 16, 2.0 ** -10, -3 * 2.0 ** -10, 5 * 2.0 ** -10]
    v = torch.zeros(1, d)
    v[0, :len(steps)] = torch.tensor(steps) * scale
    v[0, -1] = most * scale  # 381 or 1344 sixteenths: numbers of fp16
    c = R.case([0], [1], 1, nkv, d, 16, 16, kind, torch.float16, shift=0)
    c["v"], c["k"] = v.half(), v.half()  # (position 0 rotates by nothing)
    assert torch.equal(c["v"].double(), v.double())
    g = _to(c)
    _append(g)
    R.append(**c)
    assert float(c["v_scale"][int(c["table"][0, 0]), 0, 0]) == scale
    _same_cache(g, c)


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("dtype", BOTH, ids=ids)
def test_append_of_numbers_that_are_none_and_of_none(kind, dtype):
    """Infinities, NaN, zeros and the smallest numbers; a block of NaN until it begins again."""
    c = R.case([0, 4, 16, 2, 8], [3, 2, 1, 1, 8], 2, 2, 64, 16, 8, kind, dtype, seed=2)
    c["k"][0, 3] = float("inf")
    c["v"][1, 70] = NAN
    c["k"][3], c["v"][3], c["v"][4] = 0, 0, 0
    c["v"][5] = -0.0
    c["k"][5] = torch.finfo(dtype).smallest_normal * 2.0 ** -7 * torch.sign(randn((128,), seed=9)).to(dtype)
    c["v"][6, :64] = torch.finfo(dtype).max
    c["k"][6, 64:] = torch.finfo(dtype).max
    c["k_scale"][int(c["table"][3, 0]), 1, 0] = NAN
    g = _to(c)
    for _ in range(2):  # written again over itself: nothing changes
        _append(g)
        R.append(**c)
        _same_cache(g, c)
    c["lengths"][0] = g["lengths"][0] = 0
    for n in ("k", "v"):
        c[n] = randn(tuple(c[n].shape), seed=77).to(dtype)
        g[n] = c[n].to(DEV)
    _append(g)
    R.append(**c)
    _same_cache(g, c)
    assert not c["k_scale"][int(c["table"][0, 0])].isnan()[:, 0].any()


def test_append_leaves_out_what_has_no_place():
    """Rows that pass their table, pages outside the pool, tokens of no row, positions without angles, idle rows."""
    c = R.case([5, 29, 8, 3, -1, -7], [4, 3, 9, 1, 2, 1], 2, 2, 64, 16, 8, torch.int8, torch.float16, seed=3, width=2)
    c["lengths"][1] = 30
    c["table"][2, 0] = c["k_pages"].shape[0]
    c["table"][0, 0] = -1
    c["positions"][16] = len(c["cos"])  # row 3's: a key of NaN
    for n in ("q", "k", "v"):
        c[n] = torch.cat((c[n], c[n][:3]))
    c["positions"] = torch.cat((c["positions"], c["positions"][:3]))
    g = _to(c)
    _append(g)
    R.append(**c)
    _same_cache(g, c)
    assert c["k_scale"].isnan().sum() == 2
    out = int4_hip.paged_attention8(**g)
    want, mass, reach = R.attention(**c)
    _check(out, want, mass, reach, torch.float16, 32, 64)
    assert (out[-3:] == 0).all() and (out[17:20] == 0).all() and out[4:7].isnan().all() and out[16].isnan().all()


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("out", BOTH + [torch.float32], ids=ids)
@pytest.mark.parametrize("nkv,d,S,block", [(2, 64, 16, 8), (3, 128, 64, 16), (7, 64, 8, 8)])
def test_read_is_code_times_scale(kind, out, nkv, d, S, block):
    c = R.case([40, 0, 17, 3, 8, 5], [0] * 6, nkv, nkv, d, S, block, kind, torch.bfloat16, seed=6, width=40 // S + 2)
    c["table"][3, 0] = -1
    c["table"][4, 0] = c["k_pages"].shape[0] + 5
    c["k_scale"][int(c["table"][2, 0]), 0, 0] = NAN
    starts = torch.tensor([7, 0, 3, 0, 2, -1], dtype=torch.int32)
    offsets = torch.tensor([2, 35, 35, 49, 52, 58, 60], dtype=torch.int32)
    c["lengths"] = starts
    g = _to(c)
    got = int4_hip.paged_read8(*(g[n] for n in CACHE), g["table"], g["lengths"], offsets.to(DEV), 63, out)
    want = R.read(*(c[n] for n in CACHE), c["table"], starts, offsets, 63, out)
    for a, b in zip(got, want):
        assert a.dtype == out and torch.equal(torch.nan_to_num(a.cpu().float(), nan=7e7), torch.nan_to_num(b.float(), nan=7e7))
    # past the table
    starts[2] = (c["table"].shape[1] - 1) * S + 1
    got = int4_hip.paged_read8(*(g[n] for n in CACHE), g["table"], starts.to(DEV), offsets.to(DEV), 63, out)
    want = R.read(*(c[n] for n in CACHE), c["table"], starts, offsets, 63, out)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu().isnan(), b.isnan())
    assert got[0][35 + S:49].isnan().all()


def test_read_after_append_is_near_what_was_written():
    """Within half a step of the block's scale: a hundred and twenty-seventh of its largest, or a sixteenth of itself."""
    for kind in CODES:
        c = _to(R.case([0, 9], [70, 21], 2, 2, 128, 32, 32, kind, torch.bfloat16, seed=8, shift=0))
        _append(c)
        k, v = int4_hip.paged_read8(*(c[n] for n in CACHE), c["table"], c["lengths"], c["offsets"], 91, torch.float32)
        x = c["v"].float()
        err = (v - x).abs()
        if kind == torch.int8:
            assert err.max() <= 0.5001 * x.abs().max() / 127 * 2  # (a block's scale that was there may be larger)
        else:
            assert (err <= x.abs() * 2.0 ** -4 + 2.0 ** -10 * x.abs().max() / 448 * 2).all()


# ---------------------------------------------------------------- attention
CASES = [
    # (lengths, new tokens, heads, kv heads, head_dim, page size, block)
    ([0], [1], 1, 1, 64, 16, 8),
    ([1, 0, 63], [1, 1, 1], 4, 2, 64, 8, 8),
    ([127, 128, 129, 16], [1, 1, 1, 1], 8, 2, 64, 64, 16),
    ([63, 64, 65, 200], [1, 1, 1, 1], 8, 2, 128, 64, 64),
    ([5, 100, -1, 31], [1, 1, 1, 1], 6, 1, 128, 16, 16),
    ([300, 5], [1, 1], 24, 1, 64, 32, 32),
    ([30, 0, 77, 250], [5, 3, 1, 2], 8, 2, 128, 32, 8),
    ([0, 9, 60], [70, 33, 0], 4, 2, 64, 16, 8),
    ([0], [130], 6, 2, 128, 128, 64),
    ([2, -1, 0, 40], [17, 3, 1, 16], 16, 16, 64, 64, 32),
    ([10, 20], [9, 7], 33, 1, 64, 16, 16),
]


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("dtype", BOTH, ids=ids)
@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention(i, kind, dtype):
    lens, new, nh, nkv, d, S, block = CASES[i]
    _run(R.case(lens, new, nh, nkv, d, S, block, kind, dtype, seed=i), dtype)


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (8, 0), (63, 4), (64, 64), (65, 200), (500, 3), (1 << 40, 9)])
@pytest.mark.parametrize("d,S", [(64, 16), (128, 64)])
def test_window_and_sinks(window, sinks, d, S, kind):
    """Windows of one token, as long as a unit, longer than the rows; first tokens inside and outside of them."""
    c = R.case([0, 3, 150, 420, 260], [1, 7, 1, 3, 40], 4, 2, d, S, 8, kind, torch.float16, seed=window % 97, window=window,
               sinks=sinks)
    _run(c, torch.float16)


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("dtype", BOTH, ids=ids)
@pytest.mark.parametrize("nh,nkv,d,S,block", [(4, 2, 64, 16, 8), (8, 2, 128, 64, 32), (16, 1, 64, 32, 16), (17, 1, 64, 16, 16),
                                              (4, 4, 128, 64, 64), (6, 2, 64, 8, 8), (12, 1, 128, 32, 32)])
def test_steps_of_one_token(nh, nkv, d, S, block, dtype, kind):
    """Decode steps, known to be of one token a row: values of all sizes come into blocks that are begun, held and
    full; the same as the reference's, and the same bits as without that knowledge."""
    lens, sizes = [0, 7, 30, 63, -1, 100, 2000], [1.0, 0.0, 30.0, 29.0, 1e3, 1e-3, float("inf"), 1.0, 1e3, 1e4]
    c = R.case(lens, [1] * 7, nh, nkv, d, S, block, kind, dtype, seed=nh, width=2064 // S, angles=2100)
    P, table = R.pages_for([max(n, 0) + 12 for n in lens], S, 1, width=2064 // S)
    c.update(R.cache(kind, P, nkv, S, d, block, 40), table=table)
    g = _to(c)
    for step, size in enumerate(sizes):
        for n in ("q", "k", "v"):
            x = randn(tuple(c[n].shape), seed=90 + step).float()
            x = torch.where(torch.arange(7)[:, None] % 2 == 0, x, x * (1.0 if size == float("inf") else size))
            if size == float("inf") and n != "q":
                x[3, 5] = size if n == "k" else NAN
            c[n] = x.to(dtype)
            g[n] = c[n].to(DEV)
        before = {n: g[n].clone() for n in CACHE}
        out = int4_hip.paged_attention8(**g, longest=1)
        want, mass, reach = R.attention(**c)
        _same_cache(g, c)
        _check(out, want, mass, reach, dtype, 2064, d)
        two = int4_hip.paged_attention8(**dict(g, **before))
        assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(two))
        _same_cache(before, c)
        live = (c["lengths"] >= 0).int()
        for n in ("lengths", "positions"):
            c[n] = c[n] + live
            g[n] = c[n].to(DEV)


@pytest.mark.parametrize("kind", CODES, ids=ids)
def test_one_token_of_long_rows_and_windows(kind):
    for lens, window in (([9000, 50], None), ([5000, 4999, 3], 700), ([31, 32, 33, 63, 64, 65, 95, 96], 20)):
        c = R.case(lens, [1] * len(lens), 8, 2, 64, 64, 32, kind, torch.float16, seed=len(lens), window=window, sinks=5)
        g, out = _run(c, torch.float16, longest=1)
        assert torch.equal(out, int4_hip.paged_attention8(**g, longest=1))


def test_more_tokens_than_the_longest():
    """A row that has more than it may is refused, its cache left alone; no other is."""
    for longest in (1, 2):
        c = R.case([20, 33, 5], [1, 3, 1], 4, 2, 64, 16, 8, torch.int8, torch.float16, seed=3)
        g = _to(c)
        out = int4_hip.paged_attention8(**g, longest=longest)
        c["lengths"][1] = 1 << 20  # past the table: refused by the reference
        want, mass, reach = R.attention(**c)
        _check(out, want, mass, reach, torch.float16, 64, 64)
        assert out[1:4].isnan().all() and not out[[0, 4]].isnan().any()
        _same_cache(g, c)


def test_pages_that_nobody_sees_may_be_gone():
    """Behind the window a table's entries are not read: a program gives those pages back."""
    c = R.case([700, 300], [2, 1], 4, 2, 64, 16, 16, torch.int8, torch.bfloat16, seed=5, window=100, sinks=20)
    gone = [list(range(2, (701 - 100) // 16)), list(range(2, (300 - 100) // 16))]
    for b, entries in enumerate(gone):
        c["table"][b, entries] = torch.tensor([-1, 1 << 30] * 40, dtype=torch.int32)[:len(entries)]
    _, out = _run(c, torch.bfloat16)
    assert out.isfinite().all()


@pytest.mark.parametrize("rows", [70, 130, 300])
def test_many_rows(rows):
    lens = [(37 * b) % 90 - (b % 11 == 5) * 200 for b in range(rows)]
    lens = [max(n, -1) for n in lens]
    new = [(b * 7) % 4 for b in range(rows)]
    _run(R.case(lens, new, 2, 1, 64, 16, 8, torch.float8_e4m3fn, torch.float16, seed=rows), torch.float16, longest=3)


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("lens,new,nh,nkv,d", [([9000], [1], 4, 1, 64), ([6000, 10, 900], [1, 1, 1], 6, 2, 128),
                                               ([5000, 100], [3, 60], 8, 2, 64), ([4000], [1], 40, 1, 128)])
def test_long_rows_are_cut_and_joined(lens, new, nh, nkv, d, kind):
    c = R.case(lens, new, nh, nkv, d, 64, 32, kind, torch.float16, seed=len(lens))
    g, out = _run(c, torch.float16)
    again = int4_hip.paged_attention8(**g)
    assert torch.equal(out, again)  # the same bits, the cache as it was


@pytest.mark.parametrize("dtype", BOTH, ids=ids)
def test_a_dominant_token_and_scales_of_every_size(dtype):
    """Rows that one token dominates, blocks whose scales lie 2^40 apart, queries far from 1."""
    c = R.case([200, 150, 90], [1, 2, 1], 4, 2, 64, 16, 8, torch.int8, dtype, seed=12)
    c["v_scale"] *= torch.exp2(torch.linspace(-20, 20, c["v_scale"].numel())).view(c["v_scale"].shape)
    c["k_scale"] *= torch.exp2(torch.linspace(-6, 3, c["k_scale"].numel())).view(c["k_scale"].shape)
    c["q"][1] *= 8
    c["q"][2] *= 2.0 ** -10
    _run(c, dtype)


def test_scores_far_from_zero():
    """Scores of 1e5: differences decide."""
    c = R.case([60, 33], [1, 1], 2, 1, 64, 16, 8, torch.int8, torch.bfloat16, seed=13)
    c["q"] *= 2.0 ** 14
    g = _to(c)
    out = int4_hip.paged_attention8(**g).float().cpu()
    want, mass, reach = R.attention(**c)
    assert out.isfinite().all()
    # the largest score leads by far more than its error: its value, rounded
    assert (out - want.float()).abs().max() <= 2.0 ** -7 * want.abs().max()


@pytest.mark.parametrize("kind", CODES, ids=ids)
def test_what_lies_where_nobody_looks(kind):
    """Past a row's tokens and in pages of none: codes of NaN, scales of NaN and infinity; nothing of it comes out."""
    c = R.case([20, 3, 100], [2, 1, 40], 4, 2, 64, 32, 8, kind, torch.float16, seed=14)
    if kind == torch.float8_e4m3fn:
        used = R.case([20, 3, 100], [2, 1, 40], 4, 2, 64, 32, 8, kind, torch.float16, seed=14)
        for n in ("k_pages", "v_pages"):
            x = c[n].view(torch.uint8)
            keep = x.clone()
            x[:] = 0x7F
            for b, m in enumerate([22, 4, 140]):
                for i in range(m):
                    page = int(c["table"][b, i // 32])
                    x[page, :, i % 32] = keep[page, :, i % 32]
        assert used["k_pages"].float().isfinite().all()
    for n in ("k_scale", "v_scale"):
        keep = c[n].clone()
        c[n][:] = NAN
        c[n][0::2] = float("inf")
        for b, m in enumerate([22, 4, 140]):
            for i in range(0, m, 8):
                page = int(c["table"][b, i // 32])
                c[n][page, :, i % 32 // 8] = keep[page, :, i % 32 // 8]
    _, out = _run(c, torch.float16)
    assert out.isfinite().all()


def test_tokens_of_nan_reach_those_that_see_them():
    """A code of NaN in a key or value, a scale of NaN: NaN for the tokens and heads that see it, no others."""
    c = R.case([50, 50, 50, 50], [3, 3, 3, 1], 4, 2, 64, 16, 8, torch.float8_e4m3fn, torch.float16, seed=15, window=20,
               sinks=2)
    c["k_pages"].view(torch.uint8)[int(c["table"][0, 1]), 0, 15, 7] = 0x7F       # slot 31: seen by the first token alone
    c["v_pages"].view(torch.uint8)[int(c["table"][1, 2]), 1, 0, 5] = 0xFF        # slot 32: by two
    c["k_scale"][int(c["table"][2, 1]), 0, 0] = NAN                              # slots 16..23: by none
    c["v_pages"].view(torch.uint8)[int(c["table"][3, 0]), 1, 1, 60] = 0x7F       # a sink
    g, out = _run(c, torch.float16)
    nan = out.view(10, 4, 64).isnan().cpu()
    every, some = nan.all(-1), nan.any(-1)
    assert every[0].tolist() == [True, True, False, False] and not some[1:3].any()  # of a key: all elements
    assert some[3:6, 2:].all(-1).tolist() == [True, True, False] and not some[6:9].any()
    assert (nan[3:5, 2:].nonzero()[:, 2] == 5).all() and not some[3:6, :2].any()     # of a value: its own
    assert some[9].tolist() == [False, False, True, True] and (nan[9].nonzero()[:, 1] == 60).all()


def test_pages_outside_the_pool_and_rows_past_the_table():
    c = R.case([40, 40, 31, 5], [4, 4, 2, 1], 4, 2, 64, 16, 16, torch.int8, torch.bfloat16, seed=16, width=3)
    c["table"][0, 1] = c["k_pages"].shape[0]  # seen by all of row 0
    c["lengths"][1] = 45                      # 49 slots of 48
    c["table"][2, 2] = -5                     # slot 32: the second token's own
    _, out = _run(c, torch.bfloat16)
    assert out[:8].isnan().all() and out[8].isfinite().all() and out[9].isnan().all() and out[10].isfinite().all()


def test_offsets_that_pass_32_bits():
    """A pool of more than 2^31 codes: pages at its end."""
    nkv, S, d, P = 2, 64, 128, 140000  # 2.3e9 bytes each
    c = R.case([150, 70], [2, 1], 4, nkv, d, S, 32, torch.int8, torch.bfloat16, seed=17)
    n = c["k_pages"].shape[0]
    big = dict(c)
    big["table"] = torch.where(c["table"] >= 0, c["table"] + (P - n), c["table"])
    g = {k: t.to(DEV) if isinstance(t, torch.Tensor) and k not in CACHE else t for k, t in big.items()}
    for name in CACHE:
        shape = (P,) + tuple(c[name].shape[1:])
        g[name] = torch.zeros(shape, dtype=c[name].dtype, device=DEV)
        g[name][-n:] = c[name].to(DEV)
    out = int4_hip.paged_attention8(**g)
    want, mass, reach = R.attention(**c)
    _check(out, want, mass, reach, torch.bfloat16, 192, d)
    k, v = int4_hip.paged_read8(*(g[x] for x in CACHE), g["table"], g["lengths"], g["offsets"], 3, torch.float32)
    wk, wv = R.read(*(c[x] for x in CACHE), c["table"], c["lengths"], c["offsets"], 3, torch.float32)
    assert torch.equal(k.cpu(), wk) and torch.equal(v.cpu(), wv)
    _same_cache({x: g[x][-n:] for x in CACHE}, c)


def test_strided_and_misaligned_operands():
    c = R.case([20, 33], [2, 1], 4, 2, 64, 16, 8, torch.int8, torch.float16, seed=18)
    g = _to(c)
    for n in ("q", "k", "v"):
        wide = torch.full((3, g[n].shape[1] + 24), 5.0, dtype=torch.float16, device=DEV)
        wide[:, 8:-16] = g[n]
        g[n] = wide[:, 8:-16]
    odd = torch.empty(3, 257 * 2, dtype=torch.float16, device=DEV)[:, 1:257]
    odd.copy_(g["q"])
    g["q"] = odd
    for n in ("cos", "sin"):
        wide = torch.zeros(len(g[n]), 33, device=DEV)
        wide[:, 1:] = g[n]
        g[n] = wide[:, 1:]
    for n in ("positions", "lengths"):
        two = torch.stack((g[n], g[n] - 99), 1)
        g[n] = two[:, 0]
    out = int4_hip.paged_attention8(**g)
    want, mass, reach = R.attention(**c)
    _check(out, want, mass, reach, torch.float16, 64, 64)
    _same_cache(g, c)


def test_no_tokens_and_no_rows():
    c = _to(R.case([4, 0], [0, 0], 4, 2, 64, 16, 8, torch.int8, torch.float16))
    assert int4_hip.paged_attention8(**c).shape == (0, 256)
    _append(c)
    k, v = int4_hip.paged_read8(*(c[n] for n in CACHE), c["table"], c["lengths"], c["offsets"], 0)
    assert k.shape == v.shape == (0, 128)
    none = dict(_to(R.case([4], [3], 4, 2, 64, 16, 8, torch.int8, torch.float16)))
    none.update(table=none["table"][:0], lengths=none["lengths"][:0], offsets=none["offsets"][:1])
    assert (int4_hip.paged_attention8(**none) == 0).all()
    assert (int4_hip.paged_read8(*(none[n] for n in CACHE), none["table"], none["lengths"], none["offsets"], 2)[0] == 0).all()


@pytest.mark.parametrize("kind", CODES, ids=ids)
def test_captured_calls_are_replayed(kind):
    """A decode step and a few drafts in graphs of one capture stream, replayed between eager calls."""
    c = R.case([3000, 40, 7], [1, 1, 1], 8, 2, 64, 32, 16, kind, torch.bfloat16, seed=19, width=94)
    d = R.case([900, 40], [4, 2], 8, 2, 64, 32, 16, kind, torch.bfloat16, seed=20)
    g, h = _to(c), _to(d)
    start = {n: g[n].clone() for n in CACHE}
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    for x, longest in ((g, 1), (h, None)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(int4_hip.paged_attention8(**x, longest=longest))
        graphs.append(graph)
    for n in CACHE:
        g[n].copy_(start[n])
    other = _to(R.case([100], [1], 4, 2, 64, 16, 8, kind, torch.float16, seed=1))
    want, mass, reach = R.attention(**c)
    want2, mass2, reach2 = R.attention(**d)
    for _ in range(4):
        graphs[0].replay()
        int4_hip.paged_attention8(**other)
        graphs[1].replay()
        torch.cuda.synchronize()
        _check(outs[0], want, mass, reach, torch.bfloat16, 3001, 64)
        _check(outs[1], want2, mass2, reach2, torch.bfloat16, 928, 64)
        assert torch.equal(outs[0], int4_hip.paged_attention8(**g))
        _same_cache(g, c)
    # the lengths live on the GPU: a replay with others
    g["lengths"].sub_(5)
    c["lengths"] -= 5
    graphs[0].replay()
    want, mass, reach = R.attention(**c)
    _check(outs[0], want, mass, reach, torch.bfloat16, 3001, 64)


def test_two_streams_at_once():
    """Calls on two streams have a workspace each."""
    cases = [_to(R.case([4000 + 100 * i], [1], 8, 1, 64, 64, 32, torch.int8, torch.bfloat16, seed=30 + i)) for i in range(2)]
    want = [int4_hip.paged_attention8(**c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for s, c, o in zip(streams, cases, got):
            with torch.cuda.stream(s):
                o.append(int4_hip.paged_attention8(**c))
    torch.cuda.synchronize()
    for o, w in zip(got, want):
        assert all(torch.equal(x, w) for x in o)


def test_chunks_and_tokens_make_the_same_cache_as_its_parts_say():
    """A prompt in chunks, then tokens one by one, attending throughout: as the reference does it."""
    kind, new = torch.float8_e4m3fn, [20, 13, 1, 1, 4]
    c = R.case([0], [39], 4, 2, 64, 16, 16, kind, torch.float16, seed=21, shift=0)
    g, at = _to(c), 0
    for n in new:
        one = {k: (t[at:at + n] if k in ("q", "k", "v", "positions") else t) for k, t in c.items()}
        one.update(lengths=torch.tensor([at], dtype=torch.int32), offsets=torch.tensor([0, n], dtype=torch.int32))
        h = {k: (g[k] if k in CACHE or k == "table" else t) for k, t in _to(one).items()}
        out = int4_hip.paged_attention8(**h)
        want, mass, reach = R.attention(**one)
        _check(out, want, mass, reach, torch.float16, 48, 64)
        _same_cache(g, c)
        at += n


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("dtype", BOTH, ids=ids)
def test_codes_of_many_tokens(kind, dtype):
    """Against the definition on the GPU in 64 bits: enough values that some lie next to every kind of border, of
    magnitudes that reach the subnormal codes, pairs that nearly cancel, and what 32 bits cannot hold."""
    T, nkv, d, S, block = 3000, 4, 128, 64, 32
    c = _to(R.case([0], [T], nkv, nkv, d, S, block, kind, dtype, seed=23, shift=5))
    g = torch.Generator(DEV).manual_seed(3)
    for n in ("k", "v"):
        x = torch.randn((T, nkv * d), device=DEV, generator=g) * torch.exp(4 * torch.randn((T, nkv * d), device=DEV, generator=g))
        c[n] = x.clamp(-6e4, 6e4).to(dtype)
    if dtype == torch.bfloat16:
        c["k"][40] = 3e38
    c["k"][100:132], c["v"][100:132] = 1.0, 0.75  # (equal magnitudes, rotated)
    tiny = torch.finfo(dtype).smallest_normal * 2.0 ** -3  # subnormal numbers, and in bf16 the smallest scale
    for n in ("k", "v"):
        c[n][320:400] = (torch.randn((80, nkv * d), device=DEV, generator=g) * tiny).to(dtype)
    pos = c["positions"].long()
    x = c["k"].double().view(T, nkv, d)
    h, co, si = d // 2, c["cos"].double()[pos][:, None], c["sin"].double()[pos][:, None]
    key = torch.cat((x[..., :h] * co - x[..., h:] * si, x[..., h:] * co + x[..., :h] * si), -1)
    _append(c)
    k, v = int4_hip.paged_read8(*(c[n] for n in CACHE), c["table"], c["lengths"], c["offsets"], T, torch.float32)
    pages = c["table"][0].long()
    grid = torch.tensor(R._TABLE[kind][0], device=DEV, dtype=torch.float64)
    codes = torch.tensor(R._TABLE[kind][1], device=DEV)
    for got, x, scales in ((k, key, c["k_scale"]), (v, c["v"].double().view(T, nkv, d), c["v_scale"])):
        s = scales[pages].transpose(1, 2).flatten(0, 1)[:-(-T // block)]
        a = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, -T % block)).view(-1, block, nkv, d).abs().amax((1, 3))
        most = torch.full_like(a, MOST[kind])
        want = (a / most).float().clamp(min=R.TINY)
        assert torch.equal(s, torch.where(a > 0, want, 0.0))
        y = x / s.double().repeat_interleave(block, 0)[:T, :, None]
        i = torch.searchsorted(grid, y.contiguous()).clamp(1, len(grid) - 1)
        lo, hi = grid[i - 1], grid[i]
        up = (hi - y < y - lo) | ((hi - y == y - lo) & (codes[i] % 2 == 0))
        q = torch.where(up, hi, lo)
        assert torch.equal(got.view(T, nkv, d), (q * s.double().repeat_interleave(block, 0)[:T, :, None]).float())


# ---------------------------------------------------------------- rows of many new tokens (9600 columns, token and head,
# and more, in calls of 36864 and more)
PROMPTS = [
    # (lengths, new tokens, heads, kv heads, head_dim, page size, block, window, sinks)
    ([0], [160], 64, 2, 64, 16, 8, None, 0),
    ([0, 5, 40, 0], [151, 1, 150, 3], 64, 2, 64, 64, 64, None, 0),
    ([70, 0], [150, 150], 64, 4, 128, 32, 16, None, 0),
    ([130], [205], 48, 16, 64, 64, 32, 50, 0),
    ([300, 64], [170, 160], 60, 1, 128, 64, 32, 70, 5),
    ([63], [151], 64, 8, 64, 8, 8, 1, 130),
    ([0], [160], 256, 2, 64, 16, 8, None, 0),
    ([0, 5, 40, 0], [151, 1, 150, 3], 256, 2, 64, 64, 64, None, 0),
    ([70, 0], [150, 150], 256, 4, 128, 32, 16, None, 0),
    ([130], [205], 192, 16, 64, 64, 32, 50, 0),
    ([300, 64], [170, 160], 180, 1, 128, 64, 32, 70, 5),
    ([63], [151], 256, 8, 64, 8, 8, 1, 130),
]


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("dtype", BOTH, ids=ids)
@pytest.mark.parametrize("i", range(len(PROMPTS)))
def test_prompts(i, dtype, kind):
    lens, new, nh, nkv, d, S, block, window, sinks = PROMPTS[i]
    c = R.case(lens, new, nh, nkv, d, S, block, kind, dtype, seed=70 + i, window=window, sinks=sinks)
    g, out = _run(c, dtype, longest=max(new))
    assert torch.equal(out, int4_hip.paged_attention8(**g))  # the same bits


def test_prompts_that_are_no_rows():
    """Idle and refused rows of many tokens, tokens of none, pages outside the pool, positions without angles."""
    c = R.case([4, -1, 0, 9, 2], [150, 151, 152, 153, 2], 64, 2, 64, 16, 8, torch.int8, torch.float16, seed=80)
    c["lengths"][2] = 1000
    c["table"][3, 5] = -1
    c["positions"][140] = -3
    for n in ("q", "k", "v"):
        c[n] = torch.cat((c[n], c[n][:70]))
    c["positions"] = torch.cat((c["positions"], c["positions"][:70]))
    _, out = _run(c, torch.float16)
    assert (out[150:301] == 0).all() and out[301:453].isnan().all() and (out[-70:] == 0).all()
    few = int4_hip.paged_attention8(**_to(c), longest=100)  # all rows but the last have more
    live = torch.arange(678) >= 606
    live[150:301] = True
    assert few[~live.to(DEV)].isnan().all() and (few[150:301] == 0).all() and not few[606:608].isnan().any()


def test_prompts_beside_codes_of_nan():
    """Where nobody looks, and where some do."""
    lens, new = [40, 10], [150, 160]
    c = R.case(lens, new, 128, 2, 64, 32, 8, torch.float8_e4m3fn, torch.float16, seed=81, window=60, sinks=2)
    for n in ("k_pages", "v_pages"):
        x = c[n].view(torch.uint8)
        keep = x.clone()
        x[:] = 0x7F
        for b, m in enumerate(lens):
            for i in range(m + new[b]):
                page = int(c["table"][b, i // 32])
                x[page, :, i % 32] = keep[page, :, i % 32]
    _, out = _run({k: t.clone() if isinstance(t, torch.Tensor) else t for k, t in c.items()}, torch.float16)
    assert out.isfinite().all()
    c["v_pages"].view(torch.uint8)[int(c["table"][0, 0]), 0, 20, 33] = 0xFF  # slot 20: seen up to slot 79
    c["k_pages"].view(torch.uint8)[int(c["table"][1, 0]), 1, 1, 3] = 0x7F    # a sink
    _, out = _run(c, torch.float16)
    nan = out.view(310, 2, 64, 64).isnan().cpu()
    assert nan[:40, 0, :, 33].all() and not nan[40:150, 0].any() and nan[150:, 1].all() and not nan[150:, 0].any()


def test_prompts_in_a_graph():
    c = R.case([50, 7], [150, 1], 256, 2, 64, 32, 16, torch.int8, torch.bfloat16, seed=82)
    g = _to(c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = int4_hip.paged_attention8(**g, longest=150)
    want, mass, reach = R.attention(**c)
    for _ in range(3):
        graph.replay()
        eager = int4_hip.paged_attention8(**g)
        torch.cuda.synchronize()
        _check(out, want, mass, reach, torch.bfloat16, 224, 64)
        assert torch.equal(out, eager)


# ---------------------------------------------------------------- numbers of every size
FAR = [([200, 150, 90], [1, 2, 1], 4, 2, 64, 16, 8), ([700, 300], [1, 1], 6, 1, 128, 32, 16),
       ([40, 9], [152, 3], 256, 2, 64, 32, 8), ([60], [76], 512, 2, 128, 64, 16)]


@pytest.mark.parametrize("lens,new,nh,nkv,d,S,block", FAR)
def test_scales_in_any_order(lens, new, nh, nkv, d, S, block):
    """Value scales up to 2^60 apart from one block to the next: what is large often has next to no probability."""
    c = R.case(lens, new, nh, nkv, d, S, block, torch.int8, torch.bfloat16, seed=91)
    c["v_scale"] *= torch.exp2(30 * torch.sin(torch.arange(c["v_scale"].numel()) * 1.7)).view(c["v_scale"].shape)
    c["q"] *= 4
    _run(c, torch.bfloat16, longest=max(new))


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("lens,new,nh,nkv,d,S,block", FAR)
def test_the_largest_and_the_smallest_numbers(lens, new, nh, nkv, d, S, block, kind):
    """Queries of 2^100 on keys of 2^-100 and the other way round, values of 2^120 and of 2^-110."""
    for up, there in ((100, 120), (-100, -110)):
        c = R.case(lens, new, nh, nkv, d, S, block, kind, torch.bfloat16, seed=92)
        c["q"] *= 2.0 ** up
        c["k"] *= 2.0 ** -up
        c["v"] *= 2.0 ** there
        most = MOST[kind]
        c["k_scale"] = torch.full_like(c["k_scale"], 2.0 ** -up / most)
        c["v_scale"] = torch.full_like(c["v_scale"], 2.0 ** there / most)
        _run(c, torch.bfloat16, longest=max(new))


@pytest.mark.parametrize("lens,new,nh,nkv,d,S,block", FAR)
def test_queries_that_are_no_numbers(lens, new, nh, nkv, d, S, block):
    """An infinity or NaN in a head's query makes that head's output NaN, and no other's."""
    c = R.case(lens, new, nh, nkv, d, S, block, torch.int8, torch.bfloat16, seed=93)
    c["q"][0, 5] = float("inf")
    c["q"][0, d + 1] = float("nan")
    c["q"][-1, -1] = float("-inf")
    _, out = _run(c, torch.bfloat16, longest=max(new))
    nan = out.view(-1, nh, d).isnan().all(-1)
    assert nan[0, :2].all() and nan[-1, -1] and nan.sum() == 3


def test_offsets_that_decrease():
    """Rows that overlap need more tiles than the tokens are: no sense, but the call after it is as before."""
    lens = [0] * 101 + [20000]
    c = _to(R.case([20000], [1], 8, 2, 64, 64, 8, torch.int8, torch.float16, seed=94))
    want = int4_hip.paged_attention8(**c)
    bad = dict(c)
    T = 65
    for n in ("q", "k", "v", "positions"):
        bad[n] = c[n].expand(T, *c[n].shape[1:]).contiguous()
    bad["offsets"] = torch.tensor([0, 64] * 51 + [65], dtype=torch.int32, device=DEV)
    bad["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    bad["table"] = c["table"].expand(len(lens), -1).contiguous()
    for n in CACHE:
        bad[n] = c[n].clone()
    int4_hip.paged_attention8(**bad)
    for _ in range(2):
        assert torch.equal(int4_hip.paged_attention8(**c), want)


@pytest.mark.parametrize("kind", CODES, ids=ids)
@pytest.mark.parametrize("longest", [1, None])
def test_one_token_of_thousands_of_heads(kind, longest):
    """Decode steps whose single tokens are 9600 columns each, as many as a prompt's rows begin with: written and
    attended to, whether the call knows that a row has one token (one launch) or not (the prompts' kernel)."""
    c = R.case([5, 0, 17, -1, 40], [1] * 5, 9600, 600, 64, 8, 8, kind, torch.float16, seed=95)
    _run(c, torch.float16, longest=longest)
