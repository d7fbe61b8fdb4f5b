"""GPU: what the paged cache's operators and token_logprobs would lose of their operands
is refused or resolved: gradients, tangents, negated views."""
import pytest
import torch
from torch.autograd import forward_ad

import _paged_ref as R
import int4_hip
from test_gpu_paged import DEV, _to

pytestmark = pytest.mark.gpu


def _calls(dtype=torch.float16):
    """(function, arguments by name) of one call of each operator, every argument plain."""
    c = _to(R.attention_case([5, 2], 4, 2, 64, 16, dtype, seed=1))
    i = torch.zeros(2, dtype=torch.int32, device=DEV)
    append = {n: c[n] for n in ("k", "v", "cos", "sin", "k_pages", "v_pages", "table", "weight")}
    append.update(rows=i, slots=i + 1, positions=i)
    evict = {n: c[n] for n in ("k_pages", "v_pages", "weight", "table", "lengths")}
    evict.update(new_table=torch.tensor([[2], [3]], dtype=torch.int32, device=DEV), keep=4, recent=1)
    x = torch.randn(3, 40, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    score = dict(logits=x, tokens=torch.tensor([1, 0, 39], device=DEV), top=3)
    return {"attention": (int4_hip.paged_attention, c), "append": (int4_hip.paged_append, append),
            "evict": (int4_hip.paged_evict, evict), "logprobs": (int4_hip.token_logprobs, score)}


FLOATS = [("attention", n) for n in ("q", "k", "v", "cos", "sin", "k_pages", "v_pages", "weight")] + \
         [("append", n) for n in ("k", "v", "cos", "sin", "k_pages", "v_pages", "weight")] + \
         [("evict", n) for n in ("k_pages", "v_pages", "weight")] + [("logprobs", "logits")]


@pytest.mark.parametrize("op,name", FLOATS)
def test_gradients_and_tangents_are_refused(op, name):
    f, c = _calls()[op]
    f(**c)
    with pytest.raises(AssertionError, match="no_grad"):
        f(**dict(c, **{name: c[name].clone().requires_grad_()}))
    with torch.no_grad():
        f(**dict(c, **{name: c[name].clone().requires_grad_()}))
    with forward_ad.dual_level():
        f(**c)  # no tangent among them
        with torch.no_grad(), pytest.raises(AssertionError, match="tangent"):
            f(**dict(c, **{name: forward_ad.make_dual(c[name].clone(), torch.ones_like(c[name]))}))


@pytest.mark.parametrize("op,name", FLOATS + [("attention", "lengths"), ("attention", "positions"), ("append", "rows"),
                                              ("append", "slots"), ("evict", "lengths"), ("logprobs", "tokens")])
def test_negated_views_are_resolved_or_refused(op, name):
    """An operand whose memory holds the negative of its values; what is written to is refused."""
    f, c = _calls()[op]
    plain = _calls()[op][1]
    negated = torch._neg_view(c[name].neg())
    assert negated.is_neg() and negated.is_contiguous()
    c = dict(c, **{name: negated})
    if name in ("k_pages", "v_pages", "weight"):
        with pytest.raises(AssertionError):
            f(**c)
        return
    got, want = f(**c), f(**plain)
    pairs = [(got, want)] if torch.is_tensor(got) else list(zip(got, want)) if got is not None else []
    pairs += [(c[n], plain[n]) for n in ("k_pages", "v_pages", "weight") if n in c]
    for a, b in pairs:
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) if a.is_floating_point() else torch.equal(a, b)


@pytest.mark.parametrize("op,name", [("attention", "table"), ("append", "table"), ("evict", "table"),
                                     ("evict", "new_table")])
def test_negated_tables_are_refused(op, name):
    f, c = _calls()[op]
    with pytest.raises(AssertionError):
        f(**dict(c, **{name: torch._neg_view(c[name].neg())}))
