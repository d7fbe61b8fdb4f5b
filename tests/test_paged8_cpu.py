"""CPU: refusals of the 8-bit cache's entry points and of the verification, at the C
boundary (nothing is dereferenced or launched) and in Python; the tests' own reference."""
import ctypes

import pytest
import torch

import _paged8_ref as R
import int4_hip
from int4_hip import _lib

FAKE = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _cache(**kw):
    c = dict(k=256, v=256, k_scale=256, v_scale=256, table=256, pages=4, kv_heads=2, page_size=32, head_dim=64, block=16,
             rows=2, width=3, code=0, reserved=0)
    c.update(kw)
    return _lib.Paged8Cache(*[c[n] for n, _ in _lib.Paged8Cache._fields_])


BAD_CACHES = [
    (dict(head_dim=96), _lib.ERR_UNSUPPORTED, b"heads of 96"), (dict(page_size=24), _lib.ERR_UNSUPPORTED, b"pages of 24"),
    (dict(page_size=4), _lib.ERR_UNSUPPORTED, b"pages of 4"), (dict(page_size=2048), _lib.ERR_UNSUPPORTED, b"pages"),
    (dict(block=4), _lib.ERR_UNSUPPORTED, b"blocks of 4"), (dict(block=24), _lib.ERR_UNSUPPORTED, b"blocks of 24"),
    (dict(block=64), _lib.ERR_UNSUPPORTED, b"blocks of 64"), (dict(page_size=256, block=128), _lib.ERR_UNSUPPORTED, b"blocks"),
    (dict(code=2), _lib.ERR_INVALID, b"int8 or e4m3"), (dict(pages=0), _lib.ERR_INVALID, b"0 pages"),
    (dict(kv_heads=0), _lib.ERR_INVALID, b"0 heads"), (dict(rows=-1), _lib.ERR_INVALID, b"table"),
    (dict(width=0), _lib.ERR_INVALID, b"table"), (dict(width=1 << 28), _lib.ERR_INVALID, b"table"),
    (dict(k=None), _lib.ERR_INVALID, b"null"), (dict(k_scale=None), _lib.ERR_INVALID, b"null"),
    (dict(table=None), _lib.ERR_INVALID, b"null"), (dict(v=264), _lib.ERR_INVALID, b"aligned"),
    (dict(v_scale=258), _lib.ERR_INVALID, b"scales"),
]


def _append(lib, c, dtype=0, k=FAKE, stride=128, tokens=2, angles=10, cos=FAKE, lengths=FAKE):
    return lib.w4_paged8_append(c, dtype, k, FAKE, stride, 128, tokens, lengths, FAKE, FAKE, cos, FAKE, angles, None)


def _attention(lib, c, dtype=0, k=FAKE, stride=128, tokens=2, angles=10, cos=FAKE, lengths=FAKE, q=FAKE, stride_q=256,
               heads=4, longest=0, window=0, sinks=0, out=FAKE, ws=(FAKE, 1 << 40)):
    return lib.w4_paged8_attention(c, dtype, q, k, FAKE, stride_q, stride, 128, heads, tokens, longest, window, sinks,
                                   lengths, FAKE, FAKE, cos, FAKE, angles, out, *ws, None)


def _read(lib, c, dtype=0, starts=FAKE, tokens=2, k=FAKE):
    return lib.w4_paged8_read(c, dtype, starts, FAKE, tokens, k, FAKE, None)


@pytest.mark.parametrize("change,code,word", BAD_CACHES)
def test_c_abi_rejects_bad_caches(lib, change, code, word):
    for call in (_append, _attention, _read):
        assert call(lib, _cache(**change)) == code
        assert word in lib.w4_last_error(), lib.w4_last_error()


def test_c_abi_rejects_bad_arguments(lib):
    ok = _cache()
    for call in (_append, _attention, _read):
        assert call(lib, None) == _lib.ERR_INVALID
        assert call(lib, ok, dtype=3) == _lib.ERR_INVALID and b"dtype" in lib.w4_last_error()
        assert call(lib, ok, k=None) == _lib.ERR_INVALID and b"null" in lib.w4_last_error()
        assert call(lib, ok, k=ctypes.c_void_p(264)) == _lib.ERR_INVALID and b"aligned" in lib.w4_last_error()
        assert call(lib, ok, tokens=-1) == _lib.ERR_INVALID
        assert call(lib, ok, tokens=(1 << 24) + 1) == _lib.ERR_UNSUPPORTED
        assert call(lib, ok, tokens=0, k=None) == _lib.OK
    for call in (_append, _attention):
        assert call(lib, ok, dtype=2) == _lib.ERR_INVALID
        assert call(lib, ok, stride=129) == _lib.ERR_INVALID and call(lib, ok, angles=0) == _lib.ERR_INVALID
        assert call(lib, ok, cos=None) == _lib.ERR_INVALID and call(lib, ok, lengths=None) == _lib.ERR_INVALID
        assert call(lib, ok, cos=ctypes.c_void_p(260)) == _lib.ERR_INVALID
    assert _read(lib, ok, starts=None) == _lib.ERR_INVALID
    for kw in (dict(heads=3), dict(heads=0), dict(heads=2 * 257), dict(window=-1), dict(sinks=-1), dict(longest=-1),
               dict(q=None), dict(out=None), dict(stride_q=9), dict(out=ctypes.c_void_p(264))):
        assert _attention(lib, ok, **kw) == _lib.ERR_INVALID, kw
    assert _attention(lib, ok, tokens=1 << 20, heads=256) == _lib.ERR_UNSUPPORTED
    need = lib.w4_paged8_attention_workspace_bytes(2, 2, 4, 2, 64)
    assert need > 0
    for ws in ((None, 1 << 40), (FAKE, need - 1), (ctypes.c_void_p(128), 1 << 40)):
        assert _attention(lib, ok, ws=ws) == _lib.ERR_WORKSPACE
    for bad in ((-1, 2, 4, 2, 64), (2, 0, 4, 2, 64), (2, 2, 3, 2, 64), (2, 2, 0, 2, 64), (2, 1 << 40, 4, 2, 64)):
        assert lib.w4_paged8_attention_workspace_bytes(*bad) == 0


def test_calls_of_more_threads_than_a_launch_has_are_refused(lib):
    """2^24 workgroups of 256: known before anything is written."""
    big = dict(kv_heads=4096, rows=4096, page_size=8, block=8)
    for longest in (0, 1):
        assert _attention(lib, _cache(**big), tokens=4096, heads=4096, longest=longest, stride=4096 * 64,
                          stride_q=4096 * 64) == _lib.ERR_UNSUPPORTED, longest
        assert b"4096 tokens" in lib.w4_last_error()


def _verify(lib, target=FAKE, draft=FAKE, dtype=2, rows=2, drafts=3, vocab=100, strides=(400, 100, 300, 100), tokens=FAKE,
            accept=FAKE, sample=FAKE, ws=(FAKE, 1 << 30)):
    return lib.w4_verify_drafts(target, draft, dtype, rows, drafts, vocab, *strides, tokens, FAKE, accept, sample, FAKE,
                                FAKE, *ws, None)


def test_c_abi_rejects_bad_verifications(lib):
    for kw in (dict(dtype=3), dict(rows=-1), dict(drafts=-1), dict(vocab=0), dict(strides=(-1, 100, 300, 100)),
               dict(target=None), dict(tokens=None), dict(accept=None), dict(sample=None), dict(target=ctypes.c_void_p(258)),
               dict(draft=ctypes.c_void_p(257), dtype=1)):
        assert _verify(lib, **kw) == _lib.ERR_INVALID, kw
    for kw in (dict(rows=1 << 24), dict(drafts=65), dict(vocab=(1 << 22) + 1)):
        assert _verify(lib, **kw) == _lib.ERR_UNSUPPORTED, kw
    need = lib.w4_verify_drafts_workspace_bytes(2, 100)
    for ws in ((None, 1 << 30), (FAKE, need - 1), (ctypes.c_void_p(128), 1 << 30)):
        assert _verify(lib, ws=ws) == _lib.ERR_WORKSPACE
    assert _verify(lib, rows=0, target=None) == _lib.OK
    assert lib.w4_verify_drafts_workspace_bytes(0, 100) == lib.w4_verify_drafts_workspace_bytes(2, 1 << 23) == 0


def test_python_asserts():
    """On the CPU nothing of it exists."""
    c = R.case([3, 5], [1, 1], 4, 2, 64, 16, 8, torch.int8, torch.float16)
    cache = [c[n] for n in ("k_pages", "v_pages", "k_scale", "v_scale", "table")]
    with pytest.raises(AssertionError):
        int4_hip.paged_attention8(**c)
    with pytest.raises(AssertionError):
        int4_hip.paged_append8(c["k"], c["v"], c["cos"], c["sin"], *cache, c["lengths"], c["offsets"], c["positions"])
    with pytest.raises(AssertionError):
        int4_hip.paged_read8(*cache, c["lengths"], c["offsets"], 2)
    p = torch.full((2, 3, 5), 0.2)
    with pytest.raises(AssertionError):
        int4_hip.verify_drafts(p, p[:, :2], torch.zeros((2, 2), dtype=torch.int64), torch.rand(2, 2), torch.rand(2))


@pytest.mark.parametrize("kind", R.CODES)
def test_reference_rounds_as_torch_does(kind):
    """The reference's table search against torch's own conversion, where that rounds once (fp32 numbers)."""
    x = torch.cat((torch.randn(4000, generator=torch.Generator().manual_seed(1)) * 100, torch.arange(-130, 131) / 2,
                   torch.randn(2000, generator=torch.Generator().manual_seed(2)) * 0.01)).clamp(-R.MOST[kind], R.MOST[kind])
    want = x.round() if kind == torch.int8 else x.to(kind).float()
    got = torch.tensor([R.nearest(v, kind) for v in x.double().tolist()])
    assert torch.equal(got.float(), want)


def test_reference_verifies_as_the_definition_says():
    p = torch.tensor([[[0.5, 0.3, 0.2], [0.1, 0.6, 0.3]]])
    q = torch.tensor([[[0.25, 0.5, 0.25]]])
    x = torch.tensor([[1]])
    # draft 1: target 0.3, drafted 0.5: stays where the number is below 0.6
    for u, want in ((0.59, 1), (0.61, 0)):
        accepted, token = R.verify(p, q, x, torch.tensor([[u]]), torch.tensor([0.5]))
        assert accepted.item() == want
        assert token.item() == (1 if want else 0)  # of 0.1, 0.7 the half lies in 1; only token 0 has more than drafted
