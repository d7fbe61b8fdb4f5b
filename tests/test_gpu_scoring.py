"""GPU: log probabilities, entropies and alternatives (int4_hip/scoring.py) against
64-bit log softmax on the CPU."""
import math

import pytest
import torch

import int4_hip
from _synth import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
ALL = [torch.bfloat16, torch.float16, torch.float32]
# fp32 sums of up to 2^18 terms that a tree of at most 64 sequential additions per
# leaf joins (64 x 2^-24 relative: 4e-6 of the sum, so 4e-6 of its logarithm,
# absolutely), logarithm and subtraction rounded at |values| up to 40 (2^-19 = 2e-6),
# exponentials of 1e-6: together below 2e-5
TOL = 2e-5


def _reference(x, tokens, top):
    logp = torch.log_softmax(x.double(), -1)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    entropy = torch.where(logp.isnan().any(-1), math.nan, entropy)
    given = None
    if tokens is not None:
        ok = (tokens >= 0) & (tokens < x.shape[1])
        given = torch.where(ok, logp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0], math.nan)
    best = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :top]
    return given, entropy, logp.gather(1, best), best


def _near(got, want, extra=0.0):
    got = got.double().cpu()
    assert got.shape == want.shape and torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    ok = want.isfinite()
    # an fp32 result is itself rounded, twice on its way: 2^-23 of a mask's -65504 is more than TOL
    over = ((got - want).abs() - want.abs() * 2.0 ** -23)[ok]
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= TOL + extra


def _check(x, tokens, top):
    r = int4_hip.token_logprobs(x.to(DEV), None if tokens is None else tokens.to(DEV), top=top)
    given, entropy, best_p, best = _reference(x, tokens, top)
    assert torch.equal(r.top_token.cpu(), best)
    if given is None:
        assert r.logprob is None
    else:
        _near(r.logprob, given)
    _near(r.entropy, entropy, 1e-5)  # entropies add p log p of as many terms, each up to 12
    _near(r.top_logprob, best_p)
    return r


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (3, 2, 2), (2, 63, 5), (5, 64, 64), (4, 65, 0), (7, 257, 64),
                                     (2, 1023, 20), (3, 2049, 1), (1, 8191, 8), (6, 32001, 5), (2, 50257, 64),
                                     (1, 128256, 20), (9, 128256, 1), (3, 200003, 33)])
def test_random(dtype, R, V, top):
    print(f"[logprobs] {dtype} {R}x{V} top {top}", flush=True)
    x = randn((R, V), R + V, sigma=2.5, dtype=dtype)
    tokens = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(V))
    _check(x, tokens, top)
    _check(x, None, top)


@pytest.mark.parametrize("dtype", ALL)
def test_many_rows(dtype):
    x = randn((3000, 130), 1, sigma=4.0, dtype=dtype)
    _check(x, torch.arange(3000) % 130, 7)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("R,V,top", [(3, 8192, 64), (2, 6145, 64), (50, 1000, 20), (4, 300, 20), (3, 2048, 16),
                                     (3, 2049, 32), (2, 8193, 64), (2, 20000, 64)])
def test_alternatives_of_small_vocabularies(dtype, R, V, top):
    """Every group holds alternatives, or nearly every one; many candidates for few places."""
    print(f"[logprobs] {dtype} {R}x{V} top {top}", flush=True)
    x = randn((R, V), R * V, sigma=3.0, dtype=dtype)
    x[0, V // 3:] = x[0, V // 3].clone()
    x[1, ::3] = -math.inf
    _check(x, torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(V)) // 3 * 3 + 1 - V % 2, top)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("V", [100, 5000, 128256])
def test_equal_logits(dtype, V):
    """Ties everywhere: the lowest indices, in their order."""
    x = torch.zeros((4, V), dtype=dtype)
    x[1] = -3.5
    x[2, V // 2:] = 1.0
    x[3, ::7] = 2.0
    x[3, 1::7] = -0.0
    r = _check(x, torch.tensor([0, V - 1, V // 2, 3]), 64)
    assert r.top_token[0].tolist() == list(range(64))
    # two values only, the few large ones at the end
    y = torch.full((2, V), -1.0, dtype=dtype)
    y[0, -40:] = 3.0
    y[1, V // 3] = 3.0
    _check(y, torch.tensor([V - 1, 0]), 64)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("V", [70, 9000, 128256])
def test_masked_and_not_finite(dtype, V):
    x = randn((9, V), V, dtype=dtype)
    x[0, 5:] = -math.inf                 # a few allowed tokens
    x[1, :] = -math.inf                  # none
    x[2, 1:] = -math.inf                 # one
    x[3, 17] = math.inf
    x[4, 33] = math.nan
    x[5, 3] = -math.nan
    x[6, :] = torch.finfo(dtype).min     # the type's lowest value everywhere
    x[7, 4:] = torch.finfo(dtype).min    # and as a mask
    x[8, 2:] = torch.finfo(dtype).max
    tokens = torch.tensor([2, 0, 0, 17, 1, 2, 5, 3, V - 1])
    # entropy of p log p with p = 0 counts nothing: the reference's where()
    x64 = x.clone()
    r = int4_hip.token_logprobs(x.to(DEV), tokens.to(DEV), top=64)
    given, entropy, best_p, best = _reference(x64, tokens, 64)
    _near(r.logprob, given)
    _near(r.entropy, entropy, 1e-5)
    _near(r.top_logprob, best_p)
    key = torch.where(x.isnan(), math.inf, x.float())
    nan_first = torch.argsort(x.isnan().to(torch.int8), dim=-1, descending=True, stable=True)[:, :1]
    for row in range(9):
        if row in (4, 5):  # NaN above every number
            assert r.top_token[row, 0].item() == nan_first[row].item()
        else:
            assert r.top_token[row].tolist() == torch.sort(key[row], descending=True, stable=True).indices[:64].tolist()


@pytest.mark.parametrize("dtype", ALL)
def test_sorted_rows(dtype):
    """Rising and falling rows: the candidates all in one place."""
    V = 20000
    up = (torch.arange(V, dtype=torch.float32) / 64).to(dtype)
    x = torch.stack([up, up.flip(0), -up, up - up[-1]])
    _check(x, torch.tensor([0, 1, 2, V - 1]), 64)


@pytest.mark.parametrize("dtype", ALL)
def test_strided_and_misaligned_rows(dtype):
    wide = randn((5, 3001), 3, dtype=dtype)
    tokens = torch.tensor([0, 5, 2500, 1, 2])
    g = wide.to(DEV)
    for view in (lambda t: t[:, 1:2999], lambda t: t[:, 7:2600], lambda t: t[::2, 3:], lambda t: t[:, ::3],
                 lambda t: t[:1].expand(4, 3001), lambda t: t.t().contiguous().t()):
        v = view(wide)
        tok = tokens[:v.shape[0]].clamp(max=v.shape[1] - 1)
        r = int4_hip.token_logprobs(view(g), tok.to(DEV), top=9)
        given, entropy, best_p, best = _reference(v, tok, 9)
        assert torch.equal(r.top_token.cpu(), best)
        _near(r.logprob, given), _near(r.entropy, entropy, 1e-5), _near(r.top_logprob, best_p)


def test_tokens_outside_the_vocabulary():
    x = randn((4, 100), 4)
    _check(x, torch.tensor([-1, 100, -(2 ** 40), 5]), 3)


def test_offsets_past_32_bits():
    V, stride = 1000, (1 << 31) + 4096
    big = torch.empty(2 * stride + V, dtype=torch.bfloat16, device=DEV)
    view = torch.as_strided(big, (3, V), (stride, 1))
    x = randn((3, V), 5)
    view.copy_(x.to(DEV))
    r = int4_hip.token_logprobs(view, torch.tensor([1, 2, 3], device=DEV), top=4)
    given, entropy, best_p, best = _reference(x, torch.tensor([1, 2, 3]), 4)
    assert torch.equal(r.top_token.cpu(), best)
    _near(r.logprob, given), _near(r.entropy, entropy, 1e-5)


def test_repeats_and_graph():
    x = randn((6, 128256), 6, sigma=3.0).to(DEV)
    tokens = torch.arange(6, device=DEV)
    want = int4_hip.token_logprobs(x, tokens, top=10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = int4_hip.token_logprobs(x, tokens, top=10)
    for _ in range(4):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = int4_hip.token_logprobs(x, tokens, top=10)
        for a, b, c in zip(want, got, again):
            assert torch.equal(a, b) and torch.equal(a, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = int4_hip.token_logprobs(x, tokens, top=10)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, other):
        assert torch.equal(a, b)


def test_no_rows():
    r = int4_hip.token_logprobs(torch.empty((0, 10), device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), top=3)
    assert r.logprob.shape == (0,) and r.top_token.shape == (0, 3)


def test_refusals():
    x = torch.zeros((2, 10), device=DEV)
    t = torch.zeros(2, dtype=torch.int64, device=DEV)
    for args in ((x[0], None), (x.double(), None), (x, t.int()), (x, t[:1]), (x, t.cpu())):
        with pytest.raises(AssertionError):
            int4_hip.token_logprobs(*args)
    for top in (-1, 11, 65):
        with pytest.raises(AssertionError):
            int4_hip.token_logprobs(x, t, top=top)
    with pytest.raises(AssertionError):
        int4_hip.token_logprobs(x.requires_grad_(), t)
