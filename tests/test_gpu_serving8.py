"""GPU: batched decoding over the 8-bit cache (int4_hip/serving.py): its steps against the
plain statement of the attention, sliding windows whose pages go back, drafts verified."""
import pytest
import torch

import _paged8_ref as R
import int4_hip.serving as serving
from int4_hip.llama import LlamaConfig
from int4_hip.paged8 import paged_append8, paged_attention8 as int4_attention, paged_read8
from int4_hip.scoring import verify_drafts as int4_verify
from int4_hip.serving import BatchDecoder, looked_up, run
from test_gpu_serving import CFG, DEV, _decoder, _model, _prompt

pytestmark = pytest.mark.gpu
CODES = [torch.int8, torch.float8_e4m3fn]


def _plain(q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths, offsets, positions, longest=None,
           window=None, sinks=0):
    """paged_attention8 by the reference, on the CPU."""
    c = dict(q=q, k=k, v=v, cos=cos, sin=sin, k_pages=k_pages, v_pages=v_pages, k_scale=k_scale, v_scale=v_scale,
             table=table, lengths=lengths, offsets=offsets, positions=positions)
    h = {n: t.cpu().clone() for n, t in c.items()}
    out = R.attention(**h, window=window, sinks=sinks)[0]
    for n in ("k_pages", "v_pages", "k_scale", "v_scale"):
        c[n].copy_(h[n])
    return out.to(q.dtype).to(q.device)


@pytest.mark.parametrize("kind", CODES)
def test_steps_match_the_plain_attention(kind, monkeypatch):
    """Prompts, steps and drafts together.  The tolerance is that of test_rows_match_the_single_sequence_path: the
    16-bit roundings around the attention are the same; a key or value that one of them moves by a step of its own
    may move by a step of the cache, which is no more than a few of bf16's."""
    m = _model()
    made = []
    for plain in (False, True):
        monkeypatch.setattr(serving, "paged_attention8", _plain if plain else int4_attention)
        dec = _decoder(m, cache=kind, block=8, sees=30, sinks=3)
        got = []
        for row, n in enumerate((5, 40, 17)):
            r = dec.add(row, _prompt(n, n))
            got.append(r.logprob.clone())
            dec.ids[row] = 7 * row + 1  # the same tokens in both, whatever is most likely
        for i in range(4):
            r = dec.step()
            got.append(r.alternatives.top_logprob[:3].clone())
            dec.ids[:3] = torch.tensor([3, 5, 9], device=DEV) + i
        seen = []
        monkeypatch.setattr(serving, "verify_drafts", lambda p, *a: (seen.append(p.clone()), int4_verify(p, *a))[1])
        dec.verify(torch.full((4, 2), 11, device=DEV), torch.zeros(4, 2, device=DEV), torch.full((4,), 0.5, device=DEV))
        got.append(torch.log(seen[0][:3]))
        made.append(got)
    for a, b in zip(*made):
        # (the alternatives are in order; the spread of a thousand logits is about 3)
        assert (a - b).abs().max() <= 0.125 * 3.2, (a - b).abs().max()


@pytest.mark.parametrize("kind", CODES)
def test_captured_steps_are_the_eager_ones(kind):
    m = _model()
    out = []
    for capture in (False, True):
        dec = _decoder(m, cache=kind, block=16, sees=24, sinks=2)
        for row, n in enumerate((5, 40, 17)):
            dec.add(row, _prompt(n, n))
        if capture:
            dec.capture()
        out.append([dec.step().alternatives.top_logprob[:3].clone() for _ in range(20)])
        assert dec.length == [25, 60, 37, -1] and dec.lengths.tolist() == dec.length
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_pages_behind_the_window_go_back(monkeypatch):
    """Rows that outgrow the pool's pages with what they see still in it; the same bits as if all pages were kept."""
    m = _model()
    out = []
    for keeps in (True, False):
        if keeps:
            monkeypatch.setattr(BatchDecoder, "_give_back", lambda self, row: None)
        else:
            monkeypatch.undo()
        dec = _decoder(m, rows=2, pages=32 if keeps else 9, width=16, cache=torch.int8, block=16, sees=20, sinks=17)
        dec.add(0, _prompt(70, 3))
        dec.add(1, _prompt(50, 4))
        out.append([dec.step().alternatives.top_logprob.clone() for _ in range(90)])
        if not keeps:
            # of row 0's 160 slots: pages 0 and 1 hold sinks, 140.. are seen
            assert [i for i, p in enumerate(dec.owned[0]) if p is not None] == [0, 1, 8, 9]
            assert dec.table[0].tolist()[2:8] == [-1] * 6
            assert len(dec.free) == 9 - sum(p is not None for own in dec.owned for p in own)
            dec.release(0), dec.release(1)
            assert sorted(dec.free) == list(range(9))
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("kind", CODES)
def test_drafts_that_are_the_greedy_choice_stay(kind):
    """At a temperature near 0 the target is its greedy choice: drafts from a decoder that stepped there are accepted,
    up to where its two most likely tokens are nearly equal; another draft is refused and replaced."""
    m = _model()
    prompts = [_prompt(n, 60 + n) for n in (6, 30, 19)]

    def begun():
        dec = _decoder(m, cache=kind, block=8, rows=3)
        for row, p in enumerate(prompts):
            dec.add(row, p)
        return dec

    dec = begun()
    first, tokens, margins = dec.ids.clone(), [], []
    for _ in range(5):
        s = dec.step()
        tokens.append(s.token.clone())
        margins.append((s.alternatives.top_logprob[:, 0] - s.alternatives.top_logprob[:, 1]).clone())
    tokens, sure = torch.stack(tokens, 1), torch.stack(margins, 1) > 0.5
    dec = begun()
    assert torch.equal(dec.ids, first)
    high, half = torch.full((3, 4), 0.999, device=DEV), torch.full((3,), 0.5, device=DEV)
    r = dec.verify(tokens[:, :4], high, half, temperature=1e-3)
    want = sure.long().cumprod(1)[:, :4].sum(1)  # at least so many stay
    assert (r.accepted >= want).all() and sure.float().mean() > 0.5
    for row in range(3):
        n = int(r.accepted[row])
        assert dec.length[row] == len(prompts[row]) + n + 1 == dec.lengths[row] == dec.position[row]
        if sure[row, n]:
            assert r.token[row] == tokens[row, n] == dec.ids[row]
    # wrong drafts, one of them no token at all: the greedy choice instead
    dec = begun()
    wrong = (tokens[:, :2] + 1) % CFG.vocab_size
    wrong[1, 0] = 10 ** 9
    r = dec.verify(wrong, high[:, :2], half, temperature=1e-3)
    ok = sure[:, 0]
    assert (r.accepted[ok] == 0).all() and torch.equal(r.token[ok], tokens[:, 0][ok])
    # and the sequence goes on as if they had not been
    s = dec.step()
    ok = ok & sure[:, 1]
    assert torch.equal(s.token[ok], tokens[:, 1][ok])


def test_sampling_without_drafts():
    m = _model()
    dec = _decoder(m, cache=torch.int8, rows=2, block=16)
    dec.add(1, _prompt(9, 2))
    none = torch.zeros((2, 0), dtype=torch.int64, device=DEV)
    r = dec.verify(none, none.float(), torch.rand(2, device=DEV))
    assert r.accepted[1] == 0 and 0 <= int(r.token[1]) < CFG.vocab_size and dec.length == [-1, 10]
    assert dec.lengths.tolist() == [-1, 10]


def test_refusals():
    m = _model()
    for kw in (dict(cache=torch.int8, keep=8), dict(cache=torch.float16), dict(cache=torch.int8, block=24),
               dict(cache=torch.int8, block=32), dict(cache=torch.int8, block=4), dict(sees=8), dict(sinks=1),
               dict(cache=torch.int8, block=8, sees=0), dict(cache=torch.int8, block=8, sinks=-1)):
        with pytest.raises(ValueError):
            _decoder(m, **kw)
    x = torch.zeros((4, 2), dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError):
        _decoder(m).verify(x, x.float(), x[:, 0].float())
    dec = _decoder(m, cache=torch.int8, block=8, max_positions=20)
    for bad in (dict(drafts=x[:3]), dict(drafts=x[0]), dict(temperature=0.0)):
        with pytest.raises(ValueError):
            dec.verify(**{**dict(drafts=x, accept=x.float(), sample=x[:, 0].float()), **bad})
    dec.add(0, _prompt(18, 1))
    with pytest.raises(RuntimeError, match="past"):
        dec.verify(x, x.float(), x[:, 0].float())
    assert dec.length[0] == 18 and dec.evict() == []


def _state(dec):
    return [dec.k.view(torch.uint8).clone(), dec.v.view(torch.uint8).clone(), dec.scales.clone(), dec.table.clone(),
            dec.lengths.clone(), dec.positions.clone(), dec.ids.clone(), list(dec.free), [list(o) for o in dec.owned],
            list(dec.length), list(dec.position)]


def test_drafts_that_cannot_be_verified_leave_everything():
    """What the verification would refuse is refused before the drafts are in the cache."""
    m = _model()
    dec = _decoder(m, cache=torch.int8, block=8)
    dec.add(0, _prompt(15, 1))
    dec.add(2, _prompt(6, 2))
    was = _state(dec)
    x, many = (torch.zeros((4, k), dtype=torch.int64, device=DEV) for k in (2, 65))
    ok = dict(drafts=x, accept=x.float(), sample=x[:, 0].float())
    for bad in (dict(drafts=x.int()), dict(drafts=x.cpu()), dict(accept=x[:, :1].float()), dict(accept=x.double()),
                dict(accept=x.float().cpu()), dict(sample=x.float()), dict(sample=x[:, 0].half()),
                dict(sample=x[:3, 0].float()), dict(draft=torch.zeros(4, 2, CFG.vocab_size - 1, device=DEV)),
                dict(draft=torch.zeros(4, 3, CFG.vocab_size, device=DEV)),
                dict(draft=torch.zeros(4, 2, CFG.vocab_size, device=DEV, dtype=torch.bfloat16)),
                dict(draft=torch.zeros(4, 2, CFG.vocab_size)), dict(drafts=many, accept=many.float())):
        with pytest.raises((AssertionError, ValueError)):
            dec.verify(**{**ok, **bad})
        for a, b in zip(was, _state(dec)):
            assert torch.equal(a, b) if isinstance(a, torch.Tensor) else a == b


@pytest.mark.parametrize("kind", CODES)
def test_refused_drafts_leave_no_trace(kind, monkeypatch):
    """Drafts whose keys and values are far larger than those of the tokens before them, or infinite: once they are
    refused, the cache is what the accepted tokens alone make of it, bit for bit."""
    m = _model()
    dec = _decoder(m, cache=kind, block=8)
    for row, n in enumerate((5, 40, 17)):
        dec.add(row, _prompt(n, n))
    dec.ids[3] = 1
    was, K, made = _state(dec), 4, []

    def loud(q, k, v, *a, **kw):
        made.append((k.clone(), v.clone()))
        k, v = k.clone(), v.clone()
        for x in (k, v):
            x.view(4, 5, -1)[:, 1:] *= 512.0
        v.view(4, 5, -1)[2, 3] = float("inf")
        return int4_attention(q, k, v, *a, **kw)

    monkeypatch.setattr(serving, "paged_attention8", loud)
    one = torch.ones((4, K), device=DEV)  # 1 * 1 is not below any probability: refused
    r = dec.verify(torch.full((4, K), 11, device=DEV), one, one[:, 0] / 2)
    assert r.accepted.tolist()[:2] == [0, 0] and (r.token[:2] >= 0).all() and r.token[2] == -1
    # what is no number has no next token, and the row is as it was
    assert dec.length == [6, 41, 17, -1] == dec.lengths.tolist() and dec.position[:3] == [6, 41, 17]
    assert dec.ids[:2].tolist() == r.token[:2].tolist() and dec.ids[2] == was[6][2]
    lengths = torch.tensor([5, 40, -1, -1], dtype=torch.int32, device=DEV)
    starts = torch.zeros(4, dtype=torch.int32, device=DEV)
    offsets = torch.tensor([0, 6, 47, 64, 64], dtype=torch.int32, device=DEV)
    for i, (k, v) in enumerate(made):
        old = [was[0][i].view(kind), was[1][i].view(kind), was[2][0, i], was[2][1, i]]
        one = [x[::5].contiguous() for x in (k, v)]
        paged_append8(*one, dec.cos, dec.sin, *old, dec.table, lengths, dec.each, was[5])
        new = [dec.k[i], dec.v[i], dec.scales[0, i], dec.scales[1, i]]
        for a, b in zip(paged_read8(*old, dec.table, starts, offsets, 64, torch.float32),
                        paged_read8(*new, dec.table, starts, offsets, 64, torch.float32)):
            assert a.isfinite().all() and torch.equal(a, b), i
    monkeypatch.setattr(serving, "paged_attention8", int4_attention)
    assert dec.step().alternatives.top_logprob[:3].isfinite().all()


def test_a_verification_that_fails_leaves_the_tokens_as_they_were(monkeypatch):
    """An error behind the model (memory for the probabilities, for one), when the drafts are in the cache already."""
    m = _model()
    dec = _decoder(m, cache=torch.int8, block=8)
    for row, n in enumerate((5, 40, 17)):
        dec.add(row, _prompt(n, n))
    starts = torch.zeros(4, dtype=torch.int32, device=DEV)
    offsets = torch.tensor([0, 5, 45, 62, 62], dtype=torch.int32, device=DEV)

    def held():
        return [x for i in range(3) for x in paged_read8(dec.k[i], dec.v[i], dec.scales[0, i], dec.scales[1, i], dec.table,
                                                         starts, offsets, 62, torch.float32)]

    def loud(q, k, v, *a, **kw):
        return int4_attention(q, k * 512, v * 512, *a, **kw)

    def fails(*a):
        raise torch.OutOfMemoryError("none left")

    was = held(), dec.lengths.clone(), dec.ids.clone(), list(dec.length)
    monkeypatch.setattr(serving, "paged_attention8", loud)
    monkeypatch.setattr(serving, "verify_drafts", fails)
    x = torch.zeros((4, 2), dtype=torch.int64, device=DEV)
    with pytest.raises(torch.OutOfMemoryError):
        dec.verify(x, x.float(), x[:, 0].float())
    assert all(torch.equal(a, b) for a, b in zip(was[0], held()))
    assert torch.equal(was[1], dec.lengths) and torch.equal(was[2], dec.ids) and was[3] == dec.length


def test_accepted_drafts_beside_refused_ones(monkeypatch):
    """Rows that keep none, some and all of their drafts: each slot's values are within its own codes' steps of the
    keys and values that came, whatever was refused behind it."""
    m = _model()
    dec = _decoder(m, cache=torch.int8, block=16, rows=4)
    for row, n in enumerate((3, 14, 29, 7)):
        dec.add(row, _prompt(n, n))
    lengths, made = list(dec.length), []

    def seen(q, k, v, *a, **kw):
        made.append(v.clone())
        return int4_attention(q, k, v, *a, **kw)

    monkeypatch.setattr(serving, "paged_attention8", seen)
    keep = torch.tensor([[0., 0, 0], [0, 1, 1], [0, 0, 1], [1, 1, 1]], device=DEV)
    r = dec.verify(torch.full((4, 3), 11, device=DEV), keep, torch.full((4,), 0.5, device=DEV))
    assert r.accepted.tolist() == [3, 1, 2, 0]
    assert dec.length == [n + a + 1 for n, a in zip(lengths, (3, 1, 2, 0))]
    at = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    offsets = torch.tensor([0, 4, 6, 9, 10], dtype=torch.int32, device=DEV)
    take = torch.tensor([0, 1, 2, 3, 4, 5, 8, 9, 10, 12], device=DEV)
    for i, v in enumerate(made):
        got = paged_read8(dec.k[i], dec.v[i], dec.scales[0, i], dec.scales[1, i], dec.table, at, offsets, 10, torch.float32)[1]
        # half a step of the largest code's block (its scale may be twice what its values need)
        assert (got - v[take].float()).abs().max() <= dec.scales[1, i].max() * 0.5001


def test_looked_up():
    assert looked_up([1, 2, 3, 4, 2], 3) == [3, 4, 2] and looked_up([5], 2) == [5, 5]
    assert looked_up([1, 2, 2], 2) == [2, 2] and looked_up([9, 1, 9, 4, 9], 1) == [4]


def test_prompts_make_no_other_cache(monkeypatch):
    """A prompt's keys and values go into the pages and nowhere else."""
    m = _model()
    dec = _decoder(m, cache=torch.int8, block=8)
    shapes, empty = [], torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: (shapes.append(a), empty(*a, **kw))[1])
    dec.add(0, _prompt(50, 1))
    assert not [a for a in shapes if a and tuple(a[0] if isinstance(a[0], (tuple, list)) else a) in ((2, 64, 50), (2, 50, 64))]


def test_run_command():
    cfg = LlamaConfig(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64)
    for kw in (dict(cache=torch.int8), dict(cache=torch.float8_e4m3fn, sees=40, sinks=4, drafts=3)):
        r = run(batch=3, prompt_len=40, new_tokens=8, group_size=64, cfg=cfg, **kw)
        assert r["decode_tokens_per_s"] > 0 and r["cache"] == str(kw["cache"])
