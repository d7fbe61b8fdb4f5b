"""GPU: the ways through the serving operators that only large calls take, each by the
smallest call that takes it."""
import math

import pytest
import torch

import _paged_ref as R
import int4_hip
from _synth import randn
from test_gpu_paged import BOTH, _run
from test_gpu_scoring import ALL, DEV, _check as check_logprobs, _near
from test_gpu_serving import _decoder, _model, _prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ALL)
def test_logprobs_of_wide_rows_in_one_part(dtype):
    """More rows than three workgroups a CU would split: more groups a row than LDS holds."""
    R_, V = 400, 140001
    print(f"[logprobs] {dtype} {R_}x{V}", flush=True)
    x = randn((R_, V), 7, sigma=2.5, dtype=dtype)
    x[3, 100:] = -math.inf
    x[5] = 1.0
    check_logprobs(x, (torch.arange(R_) * 349) % V, 20)


def test_logprobs_of_more_rows_than_a_launch_takes():
    """Two launches for 16384 rows and more, each with its own pointers."""
    n = 16500
    x = randn((n, 70), 8, sigma=2.5, dtype=torch.bfloat16)
    check_logprobs(x, torch.arange(n) % 70, 3)


def test_logprobs_of_the_widest_vocabulary():
    """Launches of 512 rows where their groups' maxima fill the scratch memory."""
    n, V, top = 516, 1 << 22, 5
    x = torch.empty((n, V), dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(DEV).manual_seed(9)
    for row in x:
        row.copy_(torch.randn(V, device=DEV, generator=g))
    tokens = torch.arange(n, device=DEV) * 8111
    r = int4_hip.token_logprobs(x, tokens, top=top)
    for i in (0, 1, 511, 512, 515):
        logp = torch.log_softmax(x[i].double(), -1)
        best = torch.sort(x[i].float(), descending=True, stable=True).indices[:top]
        assert torch.equal(r.top_token[i], best)
        _near(r.top_logprob[i], logp[best].cpu())
        _near(r.logprob[i], logp[tokens[i]].cpu())
        _near(r.entropy[i], -(logp.exp() * logp).sum().cpu(), 1e-5)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("weights", [False, True])
def test_attention_of_more_rows_than_there_are_counters(dtype, weights):
    """Rows and heads past 16384: nothing is split, long rows neither."""
    lens = [(11 * i) % 23 - 1 for i in range(2100)]
    lens[7], lens[2099] = 700, 300
    print(f"[paged attention] {dtype} 2100 rows of 8/8x64", flush=True)
    _run(R.attention_case(lens, 8, 8, 64, 16, dtype, seed=17, weights=weights), dtype)


def test_a_long_row_depends_on_the_others_by_its_sums_alone():
    """Rows of up to four units of slots (256 of heads of 64) are one workgroup's and come out
    the same bits in every batch (test_gpu_serving.py).  Longer ones are cut by what the whole
    batch holds: their outputs may round the other way, 2^-8 of some of them in each of three
    layers, which together are under 0.7% of the logits' spread, taken four-fold for the largest
    of five."""
    m = _model()
    p = _prompt(900, 1)
    out = []
    for others in (False, True):
        dec = _decoder(m, pages=160, width=64, page_size=32, max_positions=1024)
        if others:
            dec.add(0, _prompt(1000, 2))
            dec.add(3, _prompt(700, 3))
        dec.add(2, p)
        got = []
        for i in range(8):
            dec.ids[2] = 17 * i + 1  # the same tokens whatever came out
            got.append(dec.step().alternatives.top_logprob[2].clone())
        out.append(torch.stack(got))
    m.allocate_cache(1024, torch.bfloat16, torch.device(DEV))
    spread = torch.log_softmax(m.prefill(p).float(), -1)[-1].std()
    assert ((out[0] - out[1]).abs().max() / spread).item() <= 0.028
