"""Batched decoding of the harness model (``llama.py``) over a paged key-value cache:
sequences of different lengths share one pool of pages and are decoded together, so
that each W4A16 linear of a step runs once for all rows (the library's 2..64-row
regimes); a cache that outgrows its budget keeps the tokens that were attended to.

A step of a layer is the norm, the grouped q/k/v product, ``paged_attention``, the
output product, the norm and the MLP; the logits go to ``token_logprobs``, whose most
likely token is the next one.  It is captured in a HIP graph: slots, lengths, positions
and the page table live on the GPU.

    python -m int4_hip.serving --batch 32 --prompt-len 512 --new-tokens 64
"""
from __future__ import annotations

import time
from typing import NamedTuple

import torch

from . import llama_ops
from .llama import (Attention, LlamaConfig, LlamaForCausalLM, _add_norm, _all_int4, _grouped, _plain, rope_inv_freq)
from .paged import paged_append, paged_attention, paged_evict
from .scoring import TokenLogprobs, token_logprobs


class Step(NamedTuple):
    """Of a captured step these are the graph's own tensors, and ``token`` is always ``ids``:
    the next ``step`` overwrites them, so what is to be kept is copied before it."""

    token: torch.Tensor          # int64 [rows]: the tokens now in ``ids``, idle rows' meaningless
    alternatives: TokenLogprobs  # of every row's logits


class BatchDecoder:
    """Greedy decoding of up to ``rows`` sequences at once.

    ``pages`` pages of ``page_size`` tokens are shared by all rows, at most ``width`` of
    them a row's.  With ``keep`` (and ``recent``) a row that has more than ``keep``
    tokens when ``evict`` is called is cut to its last ``recent`` and, of the others,
    those with the largest accumulated attention weight: from the last ``window`` tokens
    of its prompt, which stand for what comes next, and from every token decoded since.

    The cache holds keys and values in the model's dtype (``decode_step`` of the model
    keeps them in fp32).  With ``keep`` a step holds rows * heads * width * page_size fp32
    scores, whatever the rows hold, so ``width`` is best no more than a row may need
    (of 32 rows of 32 heads 4 MB for every 1024 tokens of it).
    """

    def __init__(self, model: LlamaForCausalLM, rows: int, pages: int, width: int, page_size: int = 64,
                 max_positions: int = 8192, keep: int | None = None, recent: int = 0, top: int = 1, window: int = 32):
        c = model.config
        self.model, self.rows, self.page_size, self.width = model, rows, page_size, width
        self.heads = c.num_attention_heads, c.num_key_value_heads, c.head_dim
        weight = model.model.embed_tokens.weight
        dev, dtype = weight.device, weight.dtype
        if dtype not in llama_ops.DTYPES or c.head_dim not in (64, 128) or not weight.is_cuda:
            raise ValueError("BatchDecoder needs a bf16 or fp16 model on the GPU with heads of 64 or 128")
        if not all(_plain(layer.self_attn, Attention) for layer in model.model.layers):
            raise ValueError("BatchDecoder stands for the model's own attention: a layer has another, or a hook on it")
        if top < 1:
            raise ValueError("the most likely token is the next one: top is at least 1")
        if window < 1:
            raise ValueError("a prompt's last token, at least, weighs the ones before it")
        if keep is not None and not (keep >= 1 and 0 <= recent <= keep):
            raise ValueError(f"a row is cut to keep >= 1 tokens, 0 to keep of them the last ones: got {keep}, {recent}")
        self.keep, self.recent, self.top, self.window = keep, recent, top, window
        nl, nkv, d = c.num_hidden_layers, c.num_key_value_heads, c.head_dim
        self.k = torch.zeros((nl, pages, nkv, page_size, d), dtype=dtype, device=dev)
        self.v = torch.zeros_like(self.k)
        self.weight = torch.zeros((nl, pages, nkv, page_size), device=dev) if keep is not None else None
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.full((rows,), -1, dtype=torch.int32, device=dev)
        self.positions = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.ids = torch.zeros(rows, dtype=torch.long, device=dev)
        ang = torch.arange(max_positions, device=dev, dtype=torch.float32)[:, None] * rope_inv_freq(c).to(dev)[None, :]
        self.cos, self.sin = ang.cos(), ang.sin()
        # the host's copy: what a row holds is known without asking the GPU
        self.free = list(range(pages))
        self.owned: list[list[int]] = [[] for _ in range(rows)]
        self.length = [-1] * rows
        self.position = [0] * rows
        self.graph = None

    # -------------------------------------------------------------- pages
    def _reserve(self, row: int, tokens: int) -> None:
        """Pages for ``tokens`` tokens of a row."""
        need = -(-tokens // self.page_size) - len(self.owned[row])
        if len(self.owned[row]) + max(need, 0) > self.width:
            raise RuntimeError(f"row {row}: {tokens} tokens are more than {self.width} pages of {self.page_size}")
        if need > len(self.free):
            raise RuntimeError(f"row {row}: {need} more pages needed, {len(self.free)} free")
        if need > 0:
            new = [self.free.pop() for _ in range(need)]
            at = len(self.owned[row])
            self.table[row, at:at + need] = torch.tensor(new, dtype=torch.int32, device=self.table.device)
            self.owned[row] += new

    def release(self, row: int) -> None:
        """Forget a sequence; the row is idle."""
        self.free += self.owned[row]
        self.owned[row], self.length[row] = [], -1
        self.lengths[row] = -1

    # -------------------------------------------------------------- the model
    def _linears(self, x, mods):
        return _grouped(x, mods) if _all_int4(mods) else [m(x) for m in mods]

    def _run(self, x, attend) -> torch.Tensor:
        """Logits of the rows ``x`` [n, hidden]; ``attend(i, q, k, v)``: the attention of layer i."""
        delta = None
        for i, layer in enumerate(self.model.model.layers):
            at, norm = layer.self_attn, layer.input_layernorm
            x, h = (x, norm(x)) if delta is None else _add_norm(x, delta, norm)
            o = at.o_proj(attend(i, *self._linears(h, (at.q_proj, at.k_proj, at.v_proj))))
            x, h = _add_norm(x, o, layer.post_attention_layernorm)
            delta = layer.mlp(h)
        return self.model.lm_head(_add_norm(x, delta, self.model.model.norm)[1])

    @torch.no_grad()
    def add(self, row: int, prompt: torch.Tensor) -> TokenLogprobs:
        """Start a sequence in an idle row with a 1-D prompt; its next token is put in
        ``ids``.  Returns the log probabilities of the prompt's own tokens 1.. (and of
        the alternatives after each of its tokens), for which it makes all of the
        prompt's logits at once."""
        T, dev = prompt.shape[0], self.ids.device
        if not 0 <= row < self.rows:
            raise ValueError(f"row {row} of {self.rows}")
        if self.length[row] >= 0 or T < 1:
            raise ValueError(f"row {row} is taken, or the prompt empty")
        if T > len(self.cos):
            raise ValueError(f"{T} tokens are more than the {len(self.cos)} positions")
        self._reserve(row, T)
        nh, nkv, d = self.heads
        kc = torch.empty((nkv, d, T), device=dev)
        vc = torch.empty((nkv, T, d), device=dev)
        cos, sin = self.cos[:T], self.sin[:T]
        slots = torch.arange(T, dtype=torch.int32, device=dev)
        rows = torch.full_like(slots, row)
        own = self.table[row:row + 1, :len(self.owned[row])]

        def attend(i, q, k, v):
            weight = None if self.weight is None else self.weight[i]
            paged_append(k, v, self.cos, self.sin, self.k[i], self.v[i], self.table, rows, slots, slots, weight)
            if weight is not None:
                # the prompt's last queries weigh what they attend to, one after the other (they share the row's
                # weights); each writes its own key and value again
                for t in range(max(T - self.window, 0), T):
                    one = slice(t, t + 1)
                    paged_attention(q[one], k[one], v[one], self.cos, self.sin, self.k[i], self.v[i], own, slots[one],
                                    slots[one], weight)
            return llama_ops.attention_prefill(q, k, v, cos, sin, kc, vc, 0, nh, nkv, d)

        logits = self._run(self.model.model.embed_tokens(prompt), attend)
        given = torch.cat([prompt[1:].to(torch.int64), torch.zeros(1, dtype=torch.int64, device=dev)])
        r = token_logprobs(logits, given, top=self.top)
        self.ids[row] = r.top_token[-1, 0]
        self.length[row], self.position[row] = T, T
        self.lengths[row] = T
        self.positions[row] = T
        return TokenLogprobs(r.logprob[:-1], r.entropy, r.top_logprob, r.top_token)

    def _step(self) -> Step:
        def attend(i, q, k, v):
            return paged_attention(q, k, v, self.cos, self.sin, self.k[i], self.v[i], self.table, self.lengths,
                                   self.positions, None if self.weight is None else self.weight[i])

        logits = self._run(self.model.model.embed_tokens(self.ids), attend)
        r = token_logprobs(logits, None, top=self.top)
        live = (self.lengths >= 0).to(torch.int32)
        self.lengths += live
        self.positions += live
        self.ids.copy_(r.top_token[:, 0])
        return Step(self.ids, r)

    @torch.no_grad()
    def capture(self) -> None:
        """Capture the step in a graph; all state is put back afterwards, also where it fails."""
        state = (self.ids, self.lengths, self.positions)
        kept = [t.clone() for t in state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        try:
            with torch.cuda.stream(side):  # workspaces; idle rows write nothing to the cache
                self.lengths.fill_(-1)
                self._step()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = self._step()
        finally:
            torch.cuda.current_stream().wait_stream(side)
            for t, was in zip(state, kept):
                t.copy_(was)
        self.graph, self.out = graph, out

    @torch.no_grad()
    def step(self) -> Step:
        """One token for every live row (its id in ``ids`` goes into the cache, the next one
        comes out)."""
        for row, n in enumerate(self.length):
            if n >= 0:
                if self.position[row] >= len(self.cos):
                    raise RuntimeError(f"row {row} is past the {len(self.cos)} positions")
                self._reserve(row, n + 1)
        if self.graph is None:
            out = self._step()
        else:
            self.graph.replay()
            out = self.out
        for row, n in enumerate(self.length):
            if n >= 0:
                self.length[row] += 1
                self.position[row] += 1
        return out

    @torch.no_grad()
    def evict(self) -> list[int]:
        """Cut every row that has more than ``keep`` tokens; the rows that were cut."""
        over = [] if self.keep is None else [r for r, n in enumerate(self.length) if n > self.keep]
        if not over:
            return over
        per = -(-self.keep // self.page_size)
        if per * len(over) > len(self.free):
            raise RuntimeError(f"{per * len(over)} pages needed to copy to, {len(self.free)} free")
        new = {r: [self.free.pop() for _ in range(per)] for r in over}
        dev = self.table.device
        to = torch.tensor([new.get(r, [-1] * per) for r in range(self.rows)], dtype=torch.int32, device=dev)
        cut = torch.tensor([r in new for r in range(self.rows)], device=dev)
        lengths = torch.where(cut, self.lengths, -1).to(torch.int32)
        for i in range(len(self.model.model.layers)):
            n = paged_evict(self.k[i], self.v[i], self.weight[i], self.table, lengths, to, self.keep, self.recent)
        self.lengths.copy_(torch.where(cut, n, self.lengths))
        full = torch.full_like(self.table, -1)
        full[:, :per] = to
        self.table.copy_(torch.where(cut[:, None], full, self.table))
        for r in over:
            self.free += self.owned[r]
            self.owned[r], self.length[r] = new[r], self.keep
        return over


@torch.no_grad()
def run(batch: int = 32, prompt_len: int = 512, new_tokens: int = 64, group_size: int = 128, seed: int = 0,
        keep: int | None = None, recent: int = 0, top: int = 5, cfg: LlamaConfig | None = None) -> dict:
    """Batched decoding of the random-init W4 model on ragged prompts: prompts put into
    the pages, then ``new_tokens`` graph-replayed steps, evicting every 64 if ``keep``."""
    from .qlinear import quantize_model_linears

    dev = torch.device("cuda")
    cfg = cfg or LlamaConfig()
    with torch.device(dev):
        model = LlamaForCausalLM(cfg)
    model.init_weights(seed)
    model = model.to(torch.bfloat16).eval()
    quantize_model_linears(model, group_size, skip=("lm_head",))
    S = 64
    width = -(-(prompt_len + new_tokens + 1) // S)
    dec = BatchDecoder(model, batch, pages=batch * width * (2 if keep is not None else 1), width=width, page_size=S,
                       max_positions=prompt_len + new_tokens + 1, keep=keep, recent=recent, top=top)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    scored = 0.0
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for row in range(batch):
        n = max(2, prompt_len * (row + 1) // batch)
        r = dec.add(row, torch.randint(0, cfg.vocab_size, (n,), device=dev, generator=g))
        scored += r.logprob.mean()
    torch.cuda.synchronize()
    prompt_s = time.perf_counter() - t0
    dec.capture()
    evicted = 0
    dec.step()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for i in range(new_tokens - 1):
        out = dec.step()
        if keep is not None and i % 64 == 63:
            evicted += len(dec.evict())
    torch.cuda.synchronize()
    s = time.perf_counter() - t0
    return {"batch": batch, "prompt_len": prompt_len, "new_tokens": new_tokens, "group_size": group_size, "keep": keep,
            "recent": recent, "rows_evicted": evicted, "prompt_s": prompt_s,
            "prompt_mean_logprob": float(scored) / batch, "decode_ms_per_step": s / (new_tokens - 1) * 1e3,
            "decode_tokens_per_s": batch * (new_tokens - 1) / s,
            "last_entropy": float(out.alternatives.entropy.mean()),
            "data": "synthetic (seeded random weights and prompts)"}


if __name__ == "__main__":
    import argparse
    import json
    ap = argparse.ArgumentParser(description="batched W4A16 decoding over a paged key-value cache (random-init model)")
    ap.add_argument("--batch", type=int, default=32)
    ap.add_argument("--prompt-len", type=int, default=512)
    ap.add_argument("--new-tokens", type=int, default=64)
    ap.add_argument("--group-size", type=int, default=128)
    ap.add_argument("--keep", type=int, default=None, help="tokens a row is cut to every 64 steps")
    ap.add_argument("--recent", type=int, default=0, help="of them, the last ones that always stay")
    a = ap.parse_args()
    print(json.dumps(run(a.batch, a.prompt_len, a.new_tokens, a.group_size, keep=a.keep, recent=a.recent)))
