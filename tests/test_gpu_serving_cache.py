"""GPU: what batched decoding (int4_hip/serving.py) does with its rows and their cache:
weights and eviction after a prompt, refusals, captures that fail."""
import math

import pytest
import torch

from _paged_ref import rope32
from test_gpu_serving import CFG, DEV, _decoder, _model, _prompt

pytestmark = pytest.mark.gpu


def _first_layer(m, dec, p):
    """(queries, keys) [T, heads, d] of the first layer, rotated in fp32, keys rounded to their type."""
    with torch.no_grad():
        layer = m.model.layers[0]
        h = layer.input_layernorm(m.model.embed_tokens(p))
        q, k = layer.self_attn.q_proj(h).cpu(), layer.self_attn.k_proj(h).cpu()
    T = len(p)
    cos, sin = dec.cos[:T, None].cpu(), dec.sin[:T, None].cpu()
    q, k = (rope32(t.float().view(T, -1, CFG.head_dim), cos, sin) for t in (q, k))
    return q, k.to(m.lm_head.weight.dtype).float()


def _row(dec, t, row, n):
    """Tokens 0..n-1 of a row of the first layer's pages ``t``: [heads, n, ..]."""
    table, j = dec.table[row].long().cpu(), torch.arange(n)
    return t[0].cpu()[table[j // dec.page_size], :, j % dec.page_size].transpose(0, 1)


@pytest.mark.parametrize("T,window", [(100, None), (100, 1), (9, None), (200, 7)])
def test_a_prompt_weighs_its_tokens(T, window):
    """After ``add`` a token's weight is the attention of the prompt's last ``window`` (32)
    queries, and an eviction right then keeps the tokens of largest weight.

    The projections are the layer's own; a probability is off by 2e-5 of itself
    (test_gpu_paged.py), a sum of up to 32 x 4 of them by as much, and by as many
    roundings of 2^-24."""
    m = _model(quantize=False)
    with torch.no_grad():
        m.model.layers[0].self_attn.q_proj.weight.mul_(8)  # attention that differs
    keep, recent = max(T // 2, 5), 3
    dec = _decoder(m, rows=2, pages=64, width=16, keep=keep, recent=recent,
                   **({} if window is None else {"window": window}))
    window = window or 32
    p = _prompt(T, T)
    dec.add(1, p)
    q, k = _first_layer(m, dec, p)
    g = q.shape[1] // k.shape[1]
    x = torch.einsum("thd,shd->hts", q.double(), k.double().repeat_interleave(g, 1)) / math.sqrt(CFG.head_dim)
    x.masked_fill_(torch.arange(T)[None, :] > torch.arange(T)[:, None], -math.inf)
    want = torch.softmax(x, -1)[:, max(T - window, 0):].sum(1).view(-1, g, T).sum(1)  # [kv heads, T]
    weight, keys = _row(dec, dec.weight, 1, T), _row(dec, dec.k, 1, T)
    assert torch.equal(keys.float(), k.transpose(0, 1))
    assert ((weight - want).abs() <= 3e-5 * want + 1e-9).all(), ((weight - want).abs() / want).max()
    assert dec.evict() == [1]
    new = _row(dec, dec.weight, 1, keep)
    keys_new = _row(dec, dec.k, 1, keep)
    for h in range(len(want)):
        kept = [i for i, w in enumerate(weight[h].tolist()) if w in set(new[h].tolist())]
        assert len(kept) == keep and kept[-recent:] == list(range(T - recent, T))
        assert torch.equal(keys_new[h], keys[h, kept])
        early = want[h, :T - recent]
        least = early.sort().values[-(keep - recent)]
        assert all((i in kept) == (w > least) for i, w in enumerate(early.tolist()) if abs(w / least - 1) > 1e-4)
    dec.step()  # and goes on


@pytest.mark.parametrize("row", [-1, -4, 4])
def test_rows_that_do_not_exist_are_refused(row):
    """A negative row is no row of the table: its tokens would go nowhere."""
    dec = _decoder(_model())
    with pytest.raises(ValueError):
        dec.add(row, _prompt(5, 1))
    assert dec.length == [-1] * 4 and len(dec.free) == 64 and dec.lengths.tolist() == dec.length


@pytest.mark.parametrize("keep,recent", [(0, 0), (-3, 0), (8, 9), (8, -1)])
def test_budgets_that_cannot_be_kept_are_refused(keep, recent):
    """When the decoder is made, and not by an eviction that has taken its pages."""
    with pytest.raises(ValueError):
        _decoder(_model(), keep=keep, recent=recent)


@pytest.mark.parametrize("at", [0, 1])
def test_a_capture_that_fails_leaves_the_rows_as_they_were(at, monkeypatch):
    """In its warm-up, or under capture: lengths, positions and tokens are put back, and
    the decoder goes on as if it had not been asked."""
    m = _model()
    out = []
    for fail in (False, True):
        dec = _decoder(m)
        dec.add(0, _prompt(20, 1))
        dec.add(2, _prompt(7, 2))
        dec.step()
        if fail:
            step, calls = dec._step, []

            def broken():
                calls.append(len(calls))
                if len(calls) == at + 1:
                    raise MemoryError("none left")
                return step()

            monkeypatch.setattr(dec, "_step", broken)
            with pytest.raises(MemoryError):
                dec.capture()
            monkeypatch.undo()
            assert dec.graph is None and dec.lengths.tolist() == dec.length
        out.append([dec.step().alternatives.top_logprob[[0, 2]].clone() for _ in range(5)])
    for a, b in zip(*out):
        assert torch.equal(a, b)
