"""GPU: batched decoding over the paged cache (int4_hip/serving.py) against the
model's own one-sequence path, and its bookkeeping of pages."""
import pytest
import torch

from int4_hip import quantize_model_linears
from int4_hip.llama import LlamaConfig, LlamaForCausalLM
from int4_hip.serving import BatchDecoder, run

pytestmark = pytest.mark.gpu
DEV = "cuda"
CFG = LlamaConfig(vocab_size=1000, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=8,
                  num_key_value_heads=2, head_dim=64)


def _model(cfg=CFG, dtype=torch.bfloat16, quantize=True, seed=0):
    with torch.device(DEV):
        m = LlamaForCausalLM(cfg)
    m.init_weights(seed)
    with torch.no_grad():
        m.lm_head.weight.mul_(10)  # logits that differ
    m = m.to(dtype).eval()
    if quantize:
        quantize_model_linears(m, 64, skip=("lm_head",))
    return m


def _prompt(n, seed, cfg=CFG):
    return torch.randint(0, cfg.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _decoder(m, **kw):
    return BatchDecoder(m, **{**dict(rows=4, pages=64, width=8, page_size=16, max_positions=256, top=5), **kw})


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("quantize", [True, False])
def test_rows_match_the_single_sequence_path(dtype, quantize):
    """Prompt log probabilities and every step's logits against prefill / decode_step.

    Both run the same kernels on the same weights up to the linears' regime (1 row or 4)
    and the cache's type: about twenty roundings to 16 bits a layer, 2^-9 of the values
    each for bf16 (2^-12 for fp16), of which some sqrt(60) = 8 add up over three layers,
    and as much again on the other side: 2^-9 * 16 = 3% of the logits' spread, taken
    four-fold for their largest of a thousand."""
    m = _model(dtype=dtype, quantize=quantize)
    tol = 0.125 if dtype is torch.bfloat16 else 0.125 / 8
    dec = _decoder(m, rows=4)
    prompts = [_prompt(n, n) for n in (5, 40, 17)]
    logits = []
    for row, p in enumerate(prompts):
        r = dec.add(row, p)
        m.allocate_cache(128, dtype, torch.device(DEV))
        want = torch.log_softmax(m.prefill(p).float(), -1)
        assert r.logprob.shape == (len(p) - 1,) and r.entropy.shape == (len(p),)
        err = (r.logprob - want[:-1].gather(1, p[1:, None])[:, 0]).abs().max() / want.std()
        assert err <= tol
        logits.append(want[-1])
    # a teacher-forced run of each sequence alone, with the tokens the batch chose
    tokens, steps = [dec.ids.clone()], []
    for _ in range(6):
        s = dec.step()
        steps.append((s.alternatives.top_token.clone(), s.alternatives.top_logprob.clone()))
        tokens.append(s.token.clone())
    for row, p in enumerate(prompts):
        m.allocate_cache(128, dtype, torch.device(DEV))
        m.prefill(p)
        for i, (top_token, top_logprob) in enumerate(steps):
            pos = torch.tensor([len(p) + i], device=DEV)
            want = torch.log_softmax(m.decode_step(tokens[i][row:row + 1], pos).float(), -1)[0]
            err = (top_logprob[row] - want[top_token[row]]).abs().max() / want.std()
            assert err <= tol, (row, i, err.item())
    assert dec.length == [11, 46, 23, -1] and dec.lengths.tolist() == dec.length


def test_a_row_does_not_depend_on_the_others():
    m = _model()
    p = _prompt(33, 1)
    out = []
    for others in (False, True):
        dec = _decoder(m)
        if others:
            dec.add(0, _prompt(50, 2))
            dec.add(3, _prompt(1, 3))
        dec.add(2, p)
        got = []
        for _ in range(20):
            s = dec.step()
            got.append((s.alternatives.top_token[2].clone(), s.alternatives.top_logprob[2].clone()))
        out.append(got)
    for a, b in zip(*out):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("page_size", [8, 64, 256])
def test_pages_do_not_change_the_result(page_size):
    m = _model()
    out = []
    for S in (16, page_size):
        dec = _decoder(m, page_size=S, width=-(-128 // S), pages=4 * -(-128 // S))
        for row in range(3):
            dec.add(row, _prompt(20 + 13 * row, row))
        out.append(torch.stack([dec.step().alternatives.top_logprob[:3].clone() for _ in range(12)]))
    assert torch.equal(*out)


def test_graph_replays_the_step():
    m = _model()
    out = []
    for graph in (False, True):
        dec = _decoder(m, keep=40, recent=8)
        for row in range(3):
            dec.add(row, _prompt(30 + row, row))
        if graph:
            dec.capture()
        got = []
        for i in range(30):
            s = dec.step()
            got.append((s.token[:3].tolist(), s.alternatives.top_logprob[:3].clone()))
            if i % 10 == 9:
                got.append((dec.evict(), dec.lengths.clone()))
        out.append(got)
    for a, b in zip(*out):
        assert a[0] == b[0] and torch.equal(a[1], b[1])


def test_eviction_frees_pages_and_keeps_going():
    m = _model()
    dec = _decoder(m, rows=2, pages=16, width=6, keep=32, recent=16)
    dec.add(0, _prompt(40, 1))
    dec.add(1, _prompt(10, 2))
    for i in range(50):
        dec.step()
        if i % 8 == 7:
            cut = dec.evict()
            assert all(dec.length[r] == 32 and len(dec.owned[r]) == 2 for r in cut)
    assert dec.lengths.tolist() == dec.length and dec.position == [90, 60]
    assert dec.positions.tolist() == dec.position
    used = sum(dec.owned, [])
    assert sorted(used + dec.free) == list(range(16)) and len(set(used)) == len(used)
    dec.release(0)
    dec.release(1)
    assert sorted(dec.free) == list(range(16)) and dec.lengths.tolist() == [-1, -1]
    # what the last 16 tokens were stays: an eviction that keeps all changes nothing but the pages
    a, b = (_decoder(m, keep=k, recent=0) for k in (64, 20))
    for d in (a, b):
        d.add(0, _prompt(20, 5))
    b.length[0] = 21  # (told to be over its budget: all 20 are copied)
    assert b.evict() == [0]
    b.length[0] = 20
    for _ in range(3):
        assert torch.equal(a.step().alternatives.top_logprob[0], b.step().alternatives.top_logprob[0])


def test_refusals():
    m = _model()
    dec = _decoder(m, pages=6, width=3, max_positions=60)
    dec.add(0, _prompt(47, 1))
    with pytest.raises(ValueError):
        dec.add(0, _prompt(3, 1))
    with pytest.raises(ValueError):
        dec.add(1, _prompt(61, 1))
    with pytest.raises(RuntimeError, match="pages"):
        dec.add(1, _prompt(49, 1))
    dec.add(1, _prompt(48, 1))
    with pytest.raises(RuntimeError, match="free|more than"):
        dec.add(2, _prompt(1, 1))
    with pytest.raises(RuntimeError):
        dec.step()
    with pytest.raises(ValueError):
        _decoder(_model(dtype=torch.float32, quantize=False))
    with pytest.raises(ValueError):
        _decoder(m, top=0)
    m.model.layers[0].self_attn.register_forward_hook(lambda *a: None)
    with pytest.raises(ValueError):
        _decoder(m)


def test_run():
    r = run(batch=3, prompt_len=40, new_tokens=70, group_size=64, keep=24, recent=8, top=2, cfg=CFG)
    assert r["rows_evicted"] == 3 and r["decode_tokens_per_s"] > 0
