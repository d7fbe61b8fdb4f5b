"""GPU: verify_drafts (int4_hip/scoring.py) against a plain statement in 64 bits."""
import pytest
import torch

import _paged8_ref as R
import int4_hip

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")


def _case(B, K, V, dtype, drafted=True, ragged=False, seed=0, near=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, K + 1, V, generator=g) * 2
    c = dict(target=torch.softmax(x, -1).to(dtype))
    draft = torch.softmax(x[:, :K] + near * torch.randn(B, K, V, generator=g), -1).to(dtype)
    c["draft"] = draft if drafted else None
    c["tokens"] = torch.multinomial(draft.float().view(B * K, V), 1, generator=g).view(B, K) if K else torch.zeros(
        B, 0, dtype=torch.int64)
    c["accept"], c["sample"] = torch.rand(B, K, generator=g), torch.rand(B, generator=g)
    c["counts"] = torch.randint(0, K + 1, (B,), generator=g).int() if ragged else None
    return c


def _run(c):
    got = int4_hip.verify_drafts(**{k: None if t is None else t.to(DEV) for k, t in c.items()})
    accepted, token = R.verify(**c)
    assert got.accepted.dtype == got.token.dtype == torch.int64
    assert torch.equal(got.accepted.cpu(), accepted), (got.accepted, accepted)
    assert torch.equal(got.token.cpu(), token), (got.token, token)
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 4, 7), (5, 2, 257), (40, 5, 1000), (2, 8, 32001), (1, 4, 128256), (9, 64, 130)])
def test_verify(B, K, V, drafted, dtype):
    _run(_case(B, K, V, dtype, drafted, ragged=B > 2, seed=B + V))


def test_no_drafts_is_sampling():
    _run(_case(6, 0, 5000, torch.float32, seed=1))
    _run(_case(6, 0, 5000, torch.float32, drafted=False, seed=2))


def test_nothing_at_once():
    c = {k: None if t is None else t.to(DEV) for k, t in _case(1, 3, 50, torch.float32).items()}
    r = int4_hip.verify_drafts(**{k: None if t is None else t[:0] for k, t in c.items()})
    assert r.accepted.shape == r.token.shape == (0,)


def test_edges_of_the_random_numbers():
    """0, the largest below 1 and what is outside; targets of one token; drafts that the target cannot have."""
    c = _case(8, 2, 300, torch.float32, seed=3)
    c["accept"][0], c["accept"][1] = 0.0, 1.0 - 2.0 ** -24
    c["sample"][0], c["sample"][1], c["sample"][2], c["sample"][3] = 0.0, 1.0 - 2.0 ** -24, 1.0, -0.5
    c["target"][4] = 0
    c["target"][4, :, 299] = 1.0
    c["tokens"][4] = 299
    c["target"][5, 0] = 0
    c["target"][5, 0, [3, 200]] = 0.5
    c["draft"][5, 0, 200] = 0.75
    c["accept"][5, 0] = 0.99
    c["target"][6, 0, int(c["tokens"][6, 0])] = 0
    c["accept"][6, 0] = 0.0  # 0 < 0 is not so: refused
    c["draft"][7, 0, int(c["tokens"][7, 0])] = 0
    c["accept"][7, 0] = 0.999
    _run(c)


def test_equal_distributions():
    """Drafts from the target itself stay, whatever the numbers; nothing to choose from without them."""
    c = _case(6, 3, 1000, torch.float32, seed=4)
    c["draft"] = c["target"][:, :3].clone()
    c["accept"][:] = 1.0 - 2.0 ** -24
    assert (_run(c).accepted == 3).all()
    # refused although no weight is left (a draft that lies outside): from the target
    c["tokens"][0, 0], c["tokens"][1, 1] = 1000, -1
    r = _run(c)
    assert r.accepted[:2].tolist() == [0, 1] and (r.token >= 0).all()


def test_no_sum_no_token():
    c = _case(7, 2, 400, torch.float32, seed=5)
    c["target"][0, :] = 0
    c["target"][1, :, 5] = NAN
    c["target"][2, :, 7] = INF
    c["target"][3, :, 9] = -0.25
    c["accept"][1:3] = 1.0  # refused
    c["draft"][1:3] = 1.0
    c["counts"] = torch.tensor([2, 2, 2, 2, -1, 3, 0], dtype=torch.int32)
    r = _run(c)
    assert r.token[:3].tolist() == [-1] * 3 and r.accepted[4:].tolist() == [-1, -1, 0] and r.token[4:6].tolist() == [-1, -1]


def test_sparse_weights():
    """Few tokens with any weight, at the ends of parts and of the vocabulary."""
    c = _case(12, 1, 9000, torch.float32, seed=6)
    c["target"][:] = 0
    for b in range(12):
        c["target"][b, :, [0, 2047, 2048, 2250 * (b % 4), 8999]] = torch.tensor([0.1, 0.2, 0.3, 0.15, 0.25])
    c["sample"] = torch.tensor([0.0, 0.0999, 0.1001, 0.29, 0.31, 0.59, 0.61, 0.74, 0.76, 0.9, 0.999, 1 - 2.0 ** -24])
    _run(c)


def test_strides():
    c = _case(4, 3, 500, torch.float16, seed=7)
    g = {k: None if t is None else t.to(DEV) for k, t in c.items()}
    wide = torch.zeros(4, 9, 700, dtype=torch.float16, device=DEV)
    wide[:, 2:6, 31:531] = g["target"]
    g["target"] = wide[:, 2:6, 31:531]
    g["draft"] = g["draft"].transpose(1, 2).contiguous().transpose(1, 2)
    g["tokens"] = g["tokens"].T.contiguous().T
    g["sample"] = torch.stack((g["sample"], g["sample"]), 1)[:, 0]
    r = int4_hip.verify_drafts(**g)
    accepted, token = R.verify(**c)
    assert torch.equal(r.accepted.cpu(), accepted) and torch.equal(r.token.cpu(), token)


def test_more_rows_than_counters():
    """Rows in slices of a launch each."""
    B = 16384 + 37
    c = _case(B, 1, 5, torch.float32, seed=8)
    _run(c)


def test_expanded_rows_and_repeats():
    c = _case(1, 4, 20000, torch.float32, seed=9)
    g = {k: None if t is None else t.to(DEV) for k, t in c.items()}
    B = 50
    for n in ("target", "draft", "tokens"):
        g[n] = g[n].expand(B, *g[n].shape[1:])
    gen = torch.Generator(DEV).manual_seed(1)
    g["accept"], g["sample"] = torch.rand(B, 4, device=DEV, generator=gen), torch.rand(B, device=DEV, generator=gen)
    r = int4_hip.verify_drafts(**g)
    accepted, token = R.verify(**{k: None if t is None else t.cpu() for k, t in g.items()})
    assert torch.equal(r.accepted.cpu(), accepted) and torch.equal(r.token.cpu(), token)
    for _ in range(3):
        s = int4_hip.verify_drafts(**g)
        assert torch.equal(r.accepted, s.accepted) and torch.equal(r.token, s.token)


def test_tokens_are_distributed_as_the_targets():
    """The point of it: what comes first after any draft has the target's probabilities (chi square, 20 degrees)."""
    V, B = 21, 40000
    g = torch.Generator(DEV).manual_seed(11)
    p = torch.softmax(torch.randn(V, device=DEV, generator=g), 0)
    q = torch.softmax(torch.randn(V, device=DEV, generator=g), 0)
    x = torch.multinomial(q, B, replacement=True, generator=g).view(B, 1)
    target = torch.stack((p, p)).expand(B, 2, V)
    r = int4_hip.verify_drafts(target, q.expand(B, 1, V), x, torch.rand(B, 1, device=DEV, generator=g),
                               torch.rand(B, device=DEV, generator=g))
    first = torch.where(r.accepted > 0, x[:, 0], r.token)
    n = torch.bincount(first, minlength=V).double()
    chi = ((n - B * p.double()) ** 2 / (B * p.double())).sum().item()
    assert chi < 60, chi  # of 20 degrees: 6e-6 of the draws are above it


def test_captured_and_replayed():
    c = _case(5, 4, 30000, torch.float32, seed=12, ragged=True)
    g = {k: None if t is None else t.to(DEV) for k, t in c.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = int4_hip.verify_drafts(**g)
    for i in range(4):
        gen = torch.Generator().manual_seed(100 + i)
        for n in ("accept", "sample"):
            c[n] = torch.rand(c[n].shape, generator=gen)
            g[n].copy_(c[n])
        graph.replay()
        s = int4_hip.verify_drafts(**g)
        accepted, token = R.verify(**c)
        assert torch.equal(r.accepted.cpu(), accepted) and torch.equal(r.token.cpu(), token)
        assert torch.equal(s.accepted.cpu(), accepted) and torch.equal(s.token.cpu(), token)
