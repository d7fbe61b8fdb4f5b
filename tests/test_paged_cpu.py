"""CPU: refusals of the paged cache's and the scoring entry points, at the C boundary
(nothing is dereferenced or launched) and in Python."""
import ctypes

import pytest
import torch

import _paged_ref as R
import int4_hip
from int4_hip import _lib

FAKE = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _cache(**kw):
    c = dict(k=256, v=256, weight=256, table=256, pages=4, kv_heads=2, page_size=16, head_dim=64, rows=2, width=3)
    c.update(kw)
    return _lib.PagedCache(*[c[n] for n, _ in _lib.PagedCache._fields_])


BAD_CACHES = [
    (dict(head_dim=96), _lib.ERR_UNSUPPORTED, b"heads of 96"), (dict(page_size=24), _lib.ERR_UNSUPPORTED, b"pages of 24"),
    (dict(page_size=4), _lib.ERR_UNSUPPORTED, b"pages of 4"), (dict(page_size=2048), _lib.ERR_UNSUPPORTED, b"pages"),
    (dict(pages=0), _lib.ERR_INVALID, b"0 pages"), (dict(kv_heads=0), _lib.ERR_INVALID, b"0 heads"),
    (dict(rows=-1), _lib.ERR_INVALID, b"table"), (dict(width=0), _lib.ERR_INVALID, b"table"),
    (dict(width=1 << 28), _lib.ERR_INVALID, b"table"), (dict(k=None), _lib.ERR_INVALID, b"null"),
    (dict(table=None), _lib.ERR_INVALID, b"null"), (dict(v=264), _lib.ERR_INVALID, b"aligned"),
]


def _append(lib, c, dtype=0, k=FAKE, stride=128, tokens=2, angles=10):
    return lib.w4_paged_append(c, dtype, k, FAKE, stride, 128, tokens, FAKE, FAKE, FAKE, FAKE, FAKE, angles, None)


def _attention(lib, c, dtype=0, q=FAKE, stride=256, heads=4, angles=10, scores=FAKE, ws=(FAKE, 1 << 40)):
    return lib.w4_paged_attention(c, dtype, q, FAKE, FAKE, stride, 128, 128, heads, FAKE, FAKE, FAKE, FAKE, angles, FAKE,
                                  scores, *ws, None)


def _evict(lib, c, dtype=0, keep=10, recent=2, width=1, scratch=FAKE):
    return lib.w4_paged_evict(c, dtype, FAKE, FAKE, width, keep, recent, scratch, FAKE, None)


@pytest.mark.parametrize("change,code,word", BAD_CACHES)
def test_c_abi_rejects_bad_caches(lib, change, code, word):
    for call in (_append, _attention, _evict):
        assert call(lib, _cache(**change)) == code
        assert word in lib.w4_last_error(), lib.w4_last_error()


def test_c_abi_rejects_bad_arguments(lib):
    ok = _cache()
    for call in (_append, _attention, _evict):
        assert call(lib, ok, dtype=2) == _lib.ERR_INVALID and b"dtype" in lib.w4_last_error()
        assert call(lib, None) == _lib.ERR_INVALID
    assert _append(lib, ok, k=None) == _lib.ERR_INVALID
    assert _append(lib, ok, k=ctypes.c_void_p(258)) == _lib.ERR_INVALID and b"aligned" in lib.w4_last_error()
    assert _append(lib, ok, stride=129) == _lib.ERR_INVALID
    assert _append(lib, ok, tokens=-1) == _lib.ERR_INVALID
    assert _append(lib, ok, angles=0) == _lib.ERR_INVALID
    assert _append(lib, ok, tokens=0) == _lib.OK
    assert _attention(lib, ok, heads=3) == _lib.ERR_INVALID and b"query heads" in lib.w4_last_error()
    assert _attention(lib, ok, heads=0) == _lib.ERR_INVALID
    assert _attention(lib, ok, q=None) == _lib.ERR_INVALID
    assert _attention(lib, ok, scores=None) == _lib.ERR_INVALID
    assert _attention(lib, ok, stride=255) == _lib.ERR_INVALID
    assert _attention(lib, _cache(rows=0)) == _lib.OK
    assert _evict(lib, ok, keep=0) == _lib.ERR_INVALID and b"keep" in lib.w4_last_error()
    assert _evict(lib, ok, keep=3, recent=4) == _lib.ERR_INVALID
    assert _evict(lib, ok, recent=-1) == _lib.ERR_INVALID
    assert _evict(lib, ok, keep=17) == _lib.ERR_INVALID
    assert _evict(lib, ok, scratch=None) == _lib.ERR_INVALID
    assert _evict(lib, _cache(weight=None)) == _lib.ERR_INVALID and b"null" in lib.w4_last_error()
    assert _evict(lib, _cache(rows=0)) == _lib.OK


def test_c_abi_rejects_bad_logits(lib):
    def call(x=FAKE, dtype=0, rows=2, vocab=100, stride=100, tokens=FAKE, top=3, logprob=FAKE, topp=FAKE):
        return lib.w4_token_logprobs(x, dtype, rows, vocab, stride, tokens, top, logprob, FAKE, topp, FAKE, FAKE,
                                     1 << 40, None)

    for bad in (dict(dtype=3), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31), dict(top=65), dict(top=-1),
                dict(vocab=2), dict(stride=-1), dict(x=None), dict(tokens=None), dict(logprob=None), dict(topp=None)):
        assert call(**bad) == _lib.ERR_INVALID, bad
        assert lib.w4_last_error()
    assert call(rows=1 << 24) == _lib.ERR_UNSUPPORTED
    assert call(rows=0) == _lib.OK


def _case():
    return R.attention_case([5, 2], 4, 2, 64, 16, torch.bfloat16, seed=1)


def test_python_refuses_cpu_tensors():
    c = _case()
    with pytest.raises(AssertionError):
        int4_hip.paged_attention(**c)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError):
        int4_hip.paged_append(c["k"], c["v"], c["cos"], c["sin"], c["k_pages"], c["v_pages"], c["table"], i, i, i)
    with pytest.raises(AssertionError):
        int4_hip.paged_evict(c["k_pages"], c["v_pages"], c["weight"], c["table"], c["lengths"], c["table"], 4, 1)
    with pytest.raises(AssertionError):
        int4_hip.token_logprobs(torch.zeros(2, 10), None)


def test_autograd_is_refused():
    c = _case()
    with pytest.raises(AssertionError, match="no_grad"):
        int4_hip.paged_attention(**dict(c, q=c["q"].requires_grad_()))
