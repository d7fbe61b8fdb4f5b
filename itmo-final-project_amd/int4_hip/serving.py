"""Batched decoding of the harness model (``llama.py``) over a paged key-value cache:
sequences of different lengths share one pool of pages and are decoded together, so
that each W4A16 linear of a step runs once for all rows (the library's 2..64-row
regimes); a cache that outgrows its budget keeps the tokens that were attended to.

A step of a layer is the norm, the grouped q/k/v product, ``paged_attention``, the
output product, the norm and the MLP; the logits go to ``token_logprobs``, whose most
likely token is the next one.  It is captured in a HIP graph: slots, lengths, positions
and the page table live on the GPU.

The cache may be held in 8 bits (``paged8.py``).  Its rows may see a sliding window and a
few first tokens only, whose other pages go back to the pool, and several drafted tokens
of every row may go through the model at once and be verified (``verify``).

    python -m int4_hip.serving --batch 32 --prompt-len 512 --new-tokens 64
    python -m int4_hip.serving --batch 8 --cache e4m3 --window 256 --sinks 4 --drafts 3
"""
from __future__ import annotations

import time
from typing import NamedTuple

import torch

from . import llama_ops
from .llama import (Attention, LlamaConfig, LlamaForCausalLM, _add_norm, _all_int4, _grouped, _plain, rope_inv_freq)
from .paged import paged_append, paged_attention, paged_evict
from .paged8 import CODES, paged_append8, paged_attention8
from .scoring import TokenLogprobs, Verified, drafts_fit, token_logprobs, verify_drafts


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

    ``cache``: ``torch.int8`` or ``torch.float8_e4m3fn`` holds it in 8 bits, with a scale for
    every ``block`` tokens of a page and head; a prompt attends to its keys and values as
    they are held.  Such a cache is not evicted from; with ``sees`` every token attends to the
    last ``sees`` tokens and the first ``sinks`` alone, and pages that no token will see
    again are given back.
    """

    def __init__(self, model: LlamaForCausalLM, rows: int, pages: int, width: int, page_size: int = 64,
                 max_positions: int = 8192, keep: int | None = None, recent: int = 0, top: int = 1, window: int = 32,
                 cache: torch.dtype | None = None, block: int = 32, sees: int | None = None, sinks: int = 0):
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
        if cache is not None and (cache not in CODES or block not in (8, 16, 32, 64) or page_size % block):
            raise ValueError("a cache of int8 or float8_e4m3fn, blocks of 8, 16, 32 or 64 tokens that fill a page: got "
                             f"{cache}, {block} of {page_size}")
        if cache is not None and keep is not None:
            raise ValueError("a cache of 8 bits is not evicted from")
        if (cache is None and (sees is not None or sinks)) or (sees is not None and sees < 1) or sinks < 0:
            raise ValueError(f"a cache of 8 bits may be seen by sees >= 1 last and sinks >= 0 first tokens: got {sees}, "
                             f"{sinks}")
        self.keep, self.recent, self.top, self.window = keep, recent, top, window
        self.sees, self.sinks = sees, sinks
        nl, nkv, d = c.num_hidden_layers, c.num_key_value_heads, c.head_dim
        self.k = torch.zeros((nl, pages, nkv, page_size, d), dtype=cache or dtype, device=dev)
        self.v = torch.zeros_like(self.k)
        self.scales = None
        if cache is not None:
            self.scales = torch.zeros((2, nl, pages, nkv, page_size // block), device=dev)
            self.each = torch.arange(rows + 1, dtype=torch.int32, device=dev)  # offsets of a token a row
        self.weight = torch.zeros((nl, pages, nkv, page_size), device=dev) if keep is not None else None
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.full((rows,), -1, dtype=torch.int32, device=dev)
        self.positions = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.ids = torch.zeros(rows, dtype=torch.long, device=dev)
        ang = torch.arange(max_positions, device=dev, dtype=torch.float32)[:, None] * rope_inv_freq(c).to(dev)[None, :]
        self.cos, self.sin = ang.cos(), ang.sin()
        # the host's copy: what a row holds is known without asking the GPU
        self.free = list(range(pages))
        self.owned: list[list[int | None]] = [[] for _ in range(rows)]  # None: given back
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
        self.free += [page for page in self.owned[row] if page is not None]
        self.owned[row], self.length[row] = [], -1
        self.lengths[row] = -1

    def _give_back(self, row: int) -> None:
        """Pages that no token will see again: behind the window of the row's next one, and no sink in them."""
        if self.sees is None:
            return
        S, own = self.page_size, self.owned[row]
        for i in range(-(-self.sinks // S), min(len(own), (self.length[row] - self.sees + 1) // S)):
            if own[i] is not None:
                self.free.append(own[i])
                own[i] = None
                self.table[row, i] = -1

    def _begun(self):
        """The blocks of a cache in 8 bits that the next tokens come into beside others, as they are: what to call to
        put them back."""
        S, n = self.page_size, self.scales.shape[-1]
        block = S // n
        at = [(self.owned[row][m // S], m % S // block) for row, m in enumerate(self.length) if m >= 0 and m % block]
        page, part = torch.tensor(at, dtype=torch.int64).view(-1, 2).T.to(self.k.device)
        # [..., pages, kv_heads, blocks of a page, words of a block]
        views = [t.view(torch.int64).view(*t.shape[:3], n, -1) for t in (self.k, self.v)] + [self.scales[..., None]]
        kept = [t[..., page, :, part, :] for t in views]

        def put_back():
            for t, was in zip(views, kept):
                t[..., page, :, part, :] = was
        return put_back

    def _write_again(self, new, starts, step, positions):
        """The first ``step`` of every row's tokens, which begin at ``starts`` of the keys and values ``new`` of the
        layers.  Layers are rows of one call; a row's other tokens are an idle row's behind it."""
        rows, T, P = self.rows, new[0][0].shape[0], self.k.shape[1]
        most = max(65535 // (2 * rows), 1)  # an operator has as many rows
        for i in range(0, len(new), most):
            n = min(most, len(new) - i)
            k, v = (torch.cat([kv[j] for kv in new[i:i + n]]) for j in range(2))
            layer = torch.arange(n, dtype=torch.int32, device=step.device)[:, None]
            real = torch.arange(2, dtype=torch.int32, device=step.device) == 0
            # (entries of no page are those of slots that no token goes to)
            table = self.table[:, None] + (layer * P)[:, None, None].expand(n, rows, 2, 1)
            lengths = torch.where(real, self.lengths[:, None], -1).expand(n, rows, 2).flatten()
            offsets = starts[:-1, None] + torch.where(real, 0, step[:, None]) + (layer * T)[..., None]
            kp, vp, ks, vs = (t[i:i + n].flatten(0, 1) for t in (self.k, self.v, *self.scales))
            paged_append8(k, v, self.cos, self.sin, kp, vp, ks, vs, table.flatten(0, 2), lengths,
                          torch.cat((offsets.flatten(), torch.full_like(starts[:1], n * T))), positions.repeat(n))

    # -------------------------------------------------------------- the model
    def _linears(self, x, mods):
        return _grouped(x, mods) if _all_int4(mods) else [m(x) for m in mods]

    def _attend8(self, table, lengths, offsets, positions, longest, new=None):
        """The attention of new tokens of the rows of ``table`` over a cache in 8 bits, for ``_run``; their keys and
        values of every layer are put into the list ``new``."""
        def attend(i, q, k, v):
            if new is not None:
                new.append((k, v))
            return paged_attention8(q, k, v, self.cos, self.sin, self.k[i], self.v[i], self.scales[0, i],
                                    self.scales[1, i], table, lengths, offsets, positions, longest=longest,
                                    window=self.sees, sinks=self.sinks)
        return attend

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
        slots = torch.arange(T, dtype=torch.int32, device=dev)
        own = self.table[row:row + 1, :len(self.owned[row])]
        if self.scales is not None:
            one = torch.tensor([0, T], dtype=torch.int32, device=dev)
            attend8 = self._attend8(own.contiguous(), one[:1], one, slots, T)
        else:
            kc = torch.empty((nkv, d, T), device=dev)
            vc = torch.empty((nkv, T, d), device=dev)
            cos, sin = self.cos[:T], self.sin[:T]
            rows = torch.full_like(slots, row)

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

        logits = self._run(self.model.model.embed_tokens(prompt), attend if self.scales is None else attend8)
        given = torch.cat([prompt[1:].to(torch.int64), torch.zeros(1, dtype=torch.int64, device=dev)])
        r = token_logprobs(logits, given, top=self.top)
        self.ids[row] = r.top_token[-1, 0]
        self.length[row], self.position[row] = T, T
        self.lengths[row] = T
        self.positions[row] = T
        self._give_back(row)
        return TokenLogprobs(r.logprob[:-1], r.entropy, r.top_logprob, r.top_token)

    def _step(self) -> Step:
        def attend(i, q, k, v):
            return paged_attention(q, k, v, self.cos, self.sin, self.k[i], self.v[i], self.table, self.lengths,
                                   self.positions, None if self.weight is None else self.weight[i])

        if self.scales is not None:
            attend = self._attend8(self.table, self.lengths, self.each, self.positions, 1)
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
                self._give_back(row)
        return out

    @torch.no_grad()
    def verify(self, drafts: torch.Tensor, accept: torch.Tensor, sample: torch.Tensor,
               draft: torch.Tensor | None = None, temperature: float = 1.0) -> Verified:
        """A step of several tokens: every live row's token in ``ids`` and its ``drafts`` int64
        [rows, K] go through the model together; those that ``verify_drafts`` accepts stay in
        the cache, and the token after them is put in ``ids``.  ``accept`` fp32 [rows, K] and
        ``sample`` fp32 [rows] are the random numbers, ``draft`` [rows, K, vocab] fp32 the
        probabilities the drafts were drawn with (None: no matter of chance).  The target's
        are the softmax of its logits over ``temperature``.

        Waits for the GPU: what the rows hold is known to the host.  Refused drafts leave no
        trace: where there are any, the blocks they came into are put back and the accepted
        tokens written to them once more.  (In the step itself all its tokens see the cache
        with the drafts in it: a draft far larger than the tokens of its block costs their
        codes bits there.)  A row whose probabilities are no numbers has the token -1 and is
        as it was before, whatever ``accepted`` says.
        """
        if self.scales is None:
            raise ValueError("drafts are verified over a cache of 8 bits")
        if drafts.dim() != 2 or drafts.shape[0] != self.rows or not temperature > 0:
            raise ValueError(f"drafts of {self.rows} rows and a temperature above 0: got {tuple(drafts.shape)}, {temperature}")
        K = drafts.shape[1]
        # (before anything of them is in the cache)
        drafts_fit((self.rows, K + 1, self.model.config.vocab_size), torch.float32, self.ids.device, draft, drafts, accept,
                   sample)
        for row, n in enumerate(self.length):
            if n >= 0:
                if self.position[row] + K >= len(self.cos):
                    raise RuntimeError(f"row {row} is past the {len(self.cos)} positions")
                self._reserve(row, n + K + 1)
        tokens = torch.cat((self.ids[:, None], drafts), 1)
        positions = (self.positions[:, None] + torch.arange(K + 1, dtype=torch.int32, device=self.ids.device)).flatten()
        put_back, new, starts = self._begun(), [], self.each * (K + 1)
        attend = self._attend8(self.table, self.lengths, starts, positions, K + 1, new)
        # (a draft outside the vocabulary is refused; until then it is some token of it)
        embed = self.model.model.embed_tokens
        try:
            logits = self._run(embed(tokens.flatten().clamp(0, embed.num_embeddings - 1)), attend)
            target = torch.softmax(logits.float() / temperature, -1).view(self.rows, K + 1, -1)
            r = verify_drafts(target, draft, drafts, accept, sample)
        except BaseException:  # (of memory, for one)
            put_back()
            raise
        good = (self.lengths >= 0) & (r.token >= 0)
        step = torch.where(good, r.accepted + 1, 0).to(torch.int32)
        steps = step.tolist()
        if any(m >= 0 and n <= K for m, n in zip(self.length, steps)):
            put_back()
            self._write_again(new, starts, step, positions)
        self.lengths += step
        self.positions += step
        self.ids.copy_(torch.where(good, r.token, self.ids))
        for row, n in enumerate(steps):
            if self.length[row] >= 0:
                self.length[row] += n
                self.position[row] += n
                self._give_back(row)
        return r

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


def looked_up(history: list[int], drafts: int) -> list[int]:
    """Drafts without a model: what followed the last token where it stood before (the last
    token itself, where it did not, and where that ends)."""
    last = history[-1]
    at = next((i for i in range(len(history) - 2, -1, -1) if history[i] == last), len(history))
    got = history[at + 1:at + 1 + drafts]
    return got + [last] * (drafts - len(got))


@torch.no_grad()
def run(batch: int = 32, prompt_len: int = 512, new_tokens: int = 64, group_size: int = 128, seed: int = 0,
        keep: int | None = None, recent: int = 0, top: int = 5, cfg: LlamaConfig | None = None,
        cache: torch.dtype | None = None, sees: int | None = None, sinks: int = 0, drafts: int = 0) -> dict:
    """Batched decoding of the random-init W4 model on ragged prompts: prompts put into
    the pages, then ``new_tokens`` graph-replayed steps, evicting every 64 if ``keep``; with
    ``drafts`` (and a ``cache`` of 8 bits) steps that verify so many looked-up tokens a row."""
    from .qlinear import quantize_model_linears

    dev = torch.device("cuda")
    cfg = cfg or LlamaConfig()
    with torch.device(dev):
        model = LlamaForCausalLM(cfg)
    model.init_weights(seed)
    model = model.to(torch.bfloat16).eval()
    quantize_model_linears(model, group_size, skip=("lm_head",))
    S = 64
    most = prompt_len + new_tokens * (drafts + 1) + 1
    width = -(-most // S)
    dec = BatchDecoder(model, batch, pages=batch * width * (2 if keep is not None else 1), width=width, page_size=S,
                       max_positions=most, keep=keep, recent=recent, top=top, cache=cache, sees=sees, sinks=sinks)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    scored, prompts = 0.0, []
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for row in range(batch):
        n = max(2, prompt_len * (row + 1) // batch)
        prompts.append(torch.randint(0, cfg.vocab_size, (n,), device=dev, generator=g))
        r = dec.add(row, prompts[-1])
        scored += r.logprob.mean()
    torch.cuda.synchronize()
    prompt_s = time.perf_counter() - t0
    result = {"batch": batch, "prompt_len": prompt_len, "new_tokens": new_tokens, "group_size": group_size, "keep": keep,
              "recent": recent, "cache": str(cache or torch.bfloat16), "sees": sees, "sinks": sinks, "drafts": drafts,
              "prompt_s": prompt_s, "prompt_mean_logprob": float(scored) / batch,
              "data": "synthetic (seeded random weights and prompts)"}
    if drafts:
        history = [p.tolist() + [t] for p, t in zip(prompts, dec.ids.tolist())]
        torch.cuda.synchronize()
        t0, made = time.perf_counter(), 0
        for _ in range(new_tokens):
            guess = torch.tensor([looked_up(h, drafts) for h in history], device=dev)
            r = dec.verify(guess, torch.rand((batch, drafts), device=dev, generator=g),
                           torch.rand(batch, device=dev, generator=g))
            for h, d, n, t in zip(history, guess.tolist(), r.accepted.tolist(), r.token.tolist()):
                if t >= 0:
                    h += d[:n] + [t]
                    made += n + 1
        s = time.perf_counter() - t0
        return {**result, "decode_ms_per_step": s / new_tokens * 1e3, "decode_tokens_per_s": made / s,
                "accepted_per_step": made / (new_tokens * batch) - 1}
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
    return {**result, "rows_evicted": evicted, "decode_ms_per_step": s / (new_tokens - 1) * 1e3,
            "decode_tokens_per_s": batch * (new_tokens - 1) / s, "last_entropy": float(out.alternatives.entropy.mean())}


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
    ap.add_argument("--cache", choices=["int8", "e4m3"], default=None, help="hold the cache in 8 bits")
    ap.add_argument("--window", type=int, default=None, help="last tokens that a token sees, of a cache in 8 bits")
    ap.add_argument("--sinks", type=int, default=0, help="first tokens that stay visible beside them")
    ap.add_argument("--drafts", type=int, default=0, help="tokens a row that a step looks up and verifies")
    a = ap.parse_args()
    cache = {None: None, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}[a.cache]
    print(json.dumps(run(a.batch, a.prompt_len, a.new_tokens, a.group_size, keep=a.keep, recent=a.recent, cache=cache,
                         sees=a.window, sinks=a.sinks, drafts=a.drafts)))
