"""GPU: what the 8-bit cache's operators and verify_drafts would lose of their operands is
refused or resolved; the native call path against the Python one; other devices' tensors."""
import pytest
import torch
from torch.autograd import forward_ad

import _paged8_ref as R
import int4_hip
from int4_hip import _lib
from test_gpu_native_path import _both, _same
from test_gpu_paged8 import CACHE, DEV, _to

pytestmark = pytest.mark.gpu


def _calls():
    """(function, arguments by name) of one call of each operator, every argument plain."""
    c = _to(R.case([5, 2], [1, 2], 4, 2, 64, 16, 8, torch.int8, torch.float16, seed=1))
    append = {n: c[n] for n in ("k", "v", "cos", "sin") + CACHE + ("table", "lengths", "offsets", "positions")}
    read = {n: c[n] for n in CACHE + ("table", "offsets")}
    read.update(starts=c["lengths"], tokens=3, dtype=torch.float16)
    g = torch.Generator(DEV).manual_seed(1)
    p = torch.softmax(torch.randn(2, 4, 50, device=DEV, generator=g), -1)
    verify = dict(target=p, draft=p[:, :3].flip(0).contiguous(), tokens=torch.zeros(2, 3, dtype=torch.int64, device=DEV),
                  accept=torch.rand(2, 3, device=DEV, generator=g), sample=torch.rand(2, device=DEV, generator=g),
                  counts=torch.tensor([3, 1], dtype=torch.int32, device=DEV))
    return {"attention": (int4_hip.paged_attention8, c), "append": (int4_hip.paged_append8, append),
            "read": (int4_hip.paged_read8, read), "verify": (int4_hip.verify_drafts, verify)}


SCALES = ("k_scale", "v_scale")
FLOATS = [("attention", n) for n in ("q", "k", "v", "cos", "sin") + SCALES] + \
         [("append", n) for n in ("k", "v", "cos", "sin") + SCALES] + [("read", n) for n in SCALES] + \
         [("verify", n) for n in ("target", "draft", "accept", "sample")]


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


@pytest.mark.parametrize("op,name", FLOATS + [("attention", "lengths"), ("attention", "offsets"), ("append", "positions"),
                                              ("read", "starts"), ("verify", "tokens"), ("verify", "counts")])
def test_negated_views_are_resolved_or_refused(op, name):
    """An operand whose memory holds the negative of its values; of the cache's it is refused."""
    f, c = _calls()[op]
    plain = _calls()[op][1]
    negated = torch._neg_view(c[name].neg())
    assert negated.is_neg()
    c = dict(c, **{name: negated})
    if name in SCALES:
        with pytest.raises(AssertionError):
            f(**c)
        return
    got, want = f(**c), f(**plain)
    pairs = [] if got is None else [(got, want)] if torch.is_tensor(got) else list(zip(got, want))
    pairs += [(c[n], plain[n]) for n in CACHE if n in c]
    for a, b in pairs:
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) if a.is_floating_point() else torch.equal(a, b)


BAD = [("attention", dict(window=0)), ("attention", dict(window=-5)), ("attention", dict(sinks=-1)),
       ("attention", dict(longest=-1)), ("read", dict(tokens=-1)), ("read", dict(dtype=torch.int8)),
       ("read", dict(dtype=torch.float64))]


@pytest.mark.parametrize("op,change", BAD)
def test_bad_numbers_are_refused(op, change):
    f, c = _calls()[op]
    with pytest.raises(AssertionError):
        f(**dict(c, **change))


@pytest.mark.parametrize("op,name", [(op, n) for op, (_, c) in (("attention", (0, ("q", "k", "v", "cos", "sin") + CACHE + (
    "table", "lengths", "offsets", "positions"))), ("read", (0, CACHE + ("table", "starts", "offsets"))),
    ("verify", (0, ("target", "draft", "tokens", "accept", "sample", "counts")))) for n in c])
def test_operands_of_another_shape_type_or_device_are_refused(op, name):
    f, c = _calls()[op]
    t = c[name]
    odd = [t.cpu(), t[:-1] if name not in ("cos", "sin", "k_pages", "v_pages") else t[..., :-1], t.double() if t.is_floating_point() else t.short()]
    for x in odd:
        with pytest.raises((AssertionError, IndexError)):
            f(**dict(c, **{name: x}))
    if name in CACHE + ("table",):
        with pytest.raises(AssertionError):
            f(**dict(c, **{name: torch.stack((t, t), -1)[..., 0]}))  # not dense


def test_scales_that_fit_no_block():
    f, c = _calls()["attention"]
    for blocks in (1, 3, 4, 16):  # pages of 16 tokens: one block is a page, four are too small
        s = torch.ones(*c["k_scale"].shape[:2], blocks, device=DEV)
        if blocks == 1:
            f(**dict(c, k_scale=s, v_scale=s.clone()))
        else:
            with pytest.raises(AssertionError):
                f(**dict(c, k_scale=s, v_scale=s.clone()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", R.CODES)
def test_call_paths_agree(kind, dtype):
    for lens, new, more in (([40, 3, -1], [1, 1, 1], dict(longest=1)), ([40, 3, 7], [3, 0, 20], dict(window=9, sinks=2))):
        c = _to(R.case(lens, new, 6, 2, 64, 16, 8, kind, dtype, seed=4))
        start = {n: c[n].clone() for n in CACHE}

        def call():
            for n in CACHE:
                c[n].copy_(start[n])
            out = int4_hip.paged_attention8(**c, **more)
            int4_hip.paged_append8(*(c[n] for n in ("k", "v", "cos", "sin") + CACHE +
                                     ("table", "lengths", "offsets", "positions")))
            kv = int4_hip.paged_read8(*(c[n] for n in CACHE), c["table"], c["lengths"], c["offsets"], 5, dtype)
            return [out.nan_to_num(3.0), *kv, *(c[n].clone() for n in CACHE)]

        _lib.load()
        assert _lib.ext.paged_attention8(*(c[n] for n in ("q", "k", "v", "cos", "sin") + CACHE + (
            "table", "lengths", "offsets", "positions")), None, None, 0) is not None
        _same(*_both(call))


def test_verification_paths_agree():
    c = _calls()["verify"][1]
    assert _lib.ext.verify_drafts(*c.values()) is not None
    for change in ({}, dict(draft=None), dict(counts=None), dict(target=c["target"].half(), draft=c["draft"].half())):
        _same(*_both(lambda: list(int4_hip.verify_drafts(**dict(c, **change)))))


def test_left_to_the_general_path():
    c = _calls()["attention"][1]
    names = ("q", "k", "v", "cos", "sin") + CACHE + ("table", "lengths", "offsets", "positions")
    rest = (None, None, 0)
    for n in names:
        odd = dict(c, **{n: c[n].cpu()})
        assert _lib.ext.paged_attention8(*(odd[m] for m in names), *rest) is None
    for rest in ((-1, None, 0), (None, 0, 0), (None, None, -1), (1.0, None, 0), (None, None, None)):
        assert _lib.ext.paged_attention8(*(c[m] for m in names), *rest) is None
    strided = dict(c, positions=torch.stack((c["positions"],) * 2, 1)[:, 0])
    assert _lib.ext.paged_attention8(*(strided[m] for m in names), None, None, 0) is None
