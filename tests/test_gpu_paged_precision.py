"""GPU: what the paged attention (int4_hip/paged.py) keeps of its operands' bits, where
it shows: rows that one token dominates, queries of every scale, results beside
infinities."""
import pytest
import torch

import _paged_ref as R
import int4_hip
from test_gpu_paged import BOTH, PROB, _check, _run, _to

pytestmark = pytest.mark.gpu


def _sink(lens, nh, nkv, d, S, dtype, gap, seed, slot=0, equal=False, weights=False):
    """Rows whose slot ``slot`` scores ``gap`` above the mean of the others (of spread 1,
    or all equal) in every head and has the value 0: the output is the others' alone."""
    c = R.attention_case(lens, nh, nkv, d, S, dtype, seed=seed, weights=weights)
    c["positions"][:] = 0  # no rotation
    B = len(lens)
    c["q"].view(B, nh, d)[:, :, 0] = 4.0
    c["k"].view(B, nkv, d)[:, :, 0] = 0.0
    c["k_pages"][..., 0] = torch.where(c["k_pages"][..., 0].isnan(), c["k_pages"][..., 0], 0.0)
    c["v"] += 1.0
    c["v_pages"] += 1.0
    if equal:
        c["k"].zero_()
        c["k_pages"].mul_(0.0)  # (NaN stays)
    for b, n in enumerate(lens):
        if n <= slot:
            continue
        p = int(c["table"][b, slot // S])
        c["k_pages"][p, :, slot % S] = 0.0
        c["k_pages"][p, :, slot % S, 0] = gap * d ** 0.5 / 4.0
        c["v_pages"][p, :, slot % S] = 0.0
    return c


# A probability enters the product in two 16-bit parts.  bf16 has fp32's range.  fp16 ends
# at 2^-24, with the largest probability of a wave's slots at 2^13 or more: what is lost of
# any other is 2^-25, a part 2^-38 of the largest, which at a gap of 18 (26 powers of two) is
# 2^-12 of the others' own, and as good as random where they differ.  So the bounds of
# rows without such a token hold: the rounding to the type, 2e-5 of the terms.
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("gap", [10.0, 14.0, 16.0, 18.0])
@pytest.mark.parametrize("lens,nh,nkv,d,S", [([300, 63, 1], 8, 2, 64, 16), ([4000], 8, 2, 64, 64),
                                             ([9000, 700], 6, 1, 128, 32), ([5000, 900], 24, 1, 64, 128)])
def test_attention_beside_a_dominant_token(dtype, gap, lens, nh, nkv, d, S):
    print(f"[paged attention] {dtype} {lens} {nh}/{nkv}x{d}, one token {gap} above", flush=True)
    for slot, equal in ((0, False), (lens[-1] // 2, False), (0, True)):
        _run(_sink(lens, nh, nkv, d, S, dtype, min(gap, 17.0) if equal else gap, seed=nh, slot=slot, equal=equal,
                   weights=slot == 0), dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("gap", [14.0, 18.0])
@pytest.mark.parametrize("nh,nkv,d", [(8, 4, 64), (16, 4, 128), (36, 4, 64)])
def test_attention_beside_a_dominant_token_many_rows(dtype, gap, nh, nkv, d):
    """Workgroups of one wave, whose slots all share the largest probability."""
    lens = [(13 * i) % 71 for i in range(140)]
    lens[3], lens[139] = 1500, 4000 * 64 // d
    print(f"[paged attention] {dtype} 140 rows of {nh}/{nkv}x{d}, one token {gap} above", flush=True)
    c = _sink(lens, nh, nkv, d, 32, dtype, gap, seed=nh)
    out = int4_hip.paged_attention(**_to(c))
    want, mass, _, _ = R.attention(**c)
    _check(out, want, mass, dtype)


# A score is a sum of d products of a query and a key of 16 bits, in 22 bits of the query and
# more: relative to |q||k| it is off by as much at every scale of the two, 2^-22, and the
# bounds of test_gpu_paged.py hold (|q||k| / sqrt(d) below 40 here too).
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("power", [-15, -8, 9, 13])
@pytest.mark.parametrize("lens,nh,nkv,d,S", [([50, 3, 700], 8, 2, 64, 16), ([900], 20, 2, 128, 64),
                                             ([5000], 24, 1, 64, 128)])
def test_attention_of_small_and_large_queries(dtype, power, lens, nh, nkv, d, S):
    """Queries of 2^power against keys of 2^-power; every other head's are 2^-4 of that."""
    print(f"[paged attention] {dtype} {lens} {nh}/{nkv}x{d}, queries of 2^{power}", flush=True)
    c = R.attention_case(lens, nh, nkv, d, S, dtype, seed=nh + power)
    B = len(lens)
    c["q"].clamp_(-3, 3).mul_(2.0 ** power).view(B, nh, d)[:, 1::2].mul_(2.0 ** -4)
    for name in ("k", "k_pages"):
        # (what fp16 holds, once rotated)
        c[name] = torch.where(c[name].isnan(), c[name], c[name].clamp(-1.3, 1.3)) * 2.0 ** -power
        c[name] = c[name].to(dtype)
    _run(c, dtype)


def test_attention_outputs_are_rounded_once():
    """bf16 outputs are the 64-bit ones rounded, but where those lie next to a boundary.

    A score of 64 products of spread 1 and its exponential are off by some 2^-22 in fp32,
    and a sum of values of either sign by as much of itself: it rounds the other way where
    it is that near to the middle of two numbers 2^-8 to 2^-7 of it apart, one in 10^4, three
    times as many with the sums that nearly cancel.  7 in 10^4 are let pass.  (Probabilities of
    16 bits give 22.)"""
    differ, count = 0, 0
    for seed in range(4):
        c = R.attention_case([1000, 900, 37, 511] * 2, 32, 8, 64, 64, torch.bfloat16, seed=100 * seed, weights=False)
        out = int4_hip.paged_attention(**_to(c)).cpu()
        want = R.attention(**c)[0].to(torch.bfloat16)
        differ += (out != want).sum().item()
        count += want.numel()
    assert differ <= 7e-4 * count, (differ, count)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("where", ["value", "key", "query", "new value", "two of them"])
@pytest.mark.parametrize("nh,nkv,d", [(8, 2, 64), (20, 2, 128), (48, 2, 64)])
def test_attention_beside_infinities(dtype, where, nh, nkv, d):
    """What is finite beside infinities and NaN, in other heads and channels and of other
    slots' weights, is as near as without them: the bounds of test_gpu_paged.py."""
    print(f"[paged attention] {dtype} {nh}/{nkv}x{d}, {where}", flush=True)
    c = R.attention_case([50, 50, 700, 50], nh, nkv, d, 16, dtype, seed=nh)
    c["q"] *= 3
    for b, bad in enumerate((float("inf"), -float("inf"), float("inf"), float("nan"))):
        p, s = int(c["table"][b, 1]), 5
        if where == "query":
            c["q"][b, 7] = bad
        elif where == "new value":
            c["v"][b, 3] = bad
        elif where == "two of them":
            c["v_pages"][p, 0, s, 40], c["v_pages"][p, 0, s + 1, 40] = bad, -bad
            c["v_pages"][p, 1, s, 11] = bad
        else:
            (c["v_pages"] if where == "value" else c["k_pages"])[p, 1, s, 9] = bad
    g = _to(c)
    out = int4_hip.paged_attention(**g)
    want, mass, _, grown = R.attention(**c)
    assert want.isfinite().any(-1).all()
    _check(out, want, mass.nan_to_num(0, 0, 0), dtype)
    got = g["weight"].double().cpu()
    assert torch.equal(got.isnan(), grown.isnan())
    ok = grown.isfinite()
    assert ((got - grown).abs()[ok] <= (PROB * nh / nkv + 2.0 ** -23 * grown.abs())[ok]).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_attention_beside_a_key_of_minus_infinity(dtype):
    """A slot that scores -inf in every head weighs nothing, and costs the others nothing."""
    c = R.attention_case([900], 8, 2, 64, 64, dtype, seed=21)
    c["positions"][:] = 0  # no rotation
    c["q"] *= 3
    c["q"].view(1, 8, 64)[:, :, 5] = c["q"].view(1, 8, 64)[:, :, 5].abs() + 0.25
    for i, s in ((0, 3), (7, 60), (13, 0)):
        c["k_pages"][int(c["table"][0, i]), :, s, 5] = -float("inf")
    _run(c, dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("size", [300.0, 3000.0, 9000.0])
@pytest.mark.parametrize("lens,nh,nkv,d", [([300, 5], 8, 2, 64), ([2000], 20, 2, 128), ([700] * 3, 24, 1, 64)])
def test_attention_of_huge_scores(dtype, size, lens, nh, nkv, d):
    """Queries and keys of up to 9000, scores of up to 5 * 10^8 (2^29 as exponents): a score
    is off by 2^-22 of that, a hundred, the two largest of some hundreds are 10^4 and more apart,
    and the output is the value of one token."""
    print(f"[paged attention] {dtype} {lens} {nh}/{nkv}x{d}, elements of {size}", flush=True)
    c = R.attention_case(lens, nh, nkv, d, 64, dtype, seed=nh + int(size))
    for name in ("q", "k", "k_pages"):
        c[name] = c[name].clamp(-4, 4) * size if name != "k_pages" else \
            torch.where(c[name].isnan(), c[name], c[name].clamp(-4, 4) * size)
    _run(c, dtype)


@pytest.mark.parametrize("size", [1e5, 1e9, 1e15])
@pytest.mark.parametrize("lens,nh,nkv,d", [([300, 5], 8, 2, 64), ([2000], 20, 2, 128), ([700] * 3, 24, 1, 64)])
def test_attention_of_scores_that_bf16_alone_has(size, lens, nh, nkv, d):
    """As above, of 10^11 to 10^31: the two largest are 10^-5 and more of that apart."""
    test_attention_of_huge_scores(torch.bfloat16, size, lens, nh, nkv, d)
