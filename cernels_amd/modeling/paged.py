"""Decoding on a paged cache: a model's decoder layers run with the library's own operators around the (swapped) experts.

The stock path keeps one cache per generate() call, in which a batch is padded to its longest sequence, and runs norm, rotary
positions, cache update and attention as separate torch operations. ``PagedDecoder`` runs the same weights on a pool of pages:
sequences of any lengths share a step without padding, prompts enter whole or in chunks, and a layer is the library's layer norm
(north_mini_code), one launch that turns queries and keys and writes keys and values to their pages, and paged attention with the
layer's window; projections, routers, experts and (deepseek_ocr_2) RMS norms stay the model's modules, with whatever swap is
installed.

    decoder = PagedDecoder(model, pages=512)
    tokens = decoder.generate([ids_a, ids_b], 64)        # greedy
    logits = decoder.step([chunk_a, chunk_b])            # or step by step: the logits behind each sequence's last token
"""

from __future__ import annotations

import statistics

import torch

from cernels_amd import ops

PAGE_SIZE = 64


class PagePool:
    """The pages of every layer, and which of them each sequence has. Page ids are shared by the layers: page 7 of a sequence is page 7
    in every layer's pool."""

    def __init__(self, layers: int, pages: int, kv_heads: int, dim: int, dtype, device, page_size: int = PAGE_SIZE):
        self.page_size, self.device = page_size, device
        self.k, self.v = ([torch.empty(pages, page_size, kv_heads, dim, dtype=dtype, device=device) for _ in range(layers)]
                          for _ in range(2))
        self.free = list(range(pages - 1, -1, -1))
        self.held: list[list[int]] = []   # per sequence
        self.counts: list[int] = []       # tokens per sequence
        self.table = torch.empty(0, 0, dtype=torch.int32, device=device)

    def open(self, sequences: int) -> None:
        """Starts over with that many empty sequences."""
        for pages in self.held:
            self.free.extend(reversed(pages))
        self.held, self.counts = [[] for _ in range(sequences)], [0] * sequences
        self.table = torch.full((sequences, 1), -1, dtype=torch.int32, device=self.device)

    def grow(self, new: list[int]) -> None:
        """Makes room for new[b] more tokens of each sequence b and counts them. Nothing changes if the pool has too few pages."""
        counts = [c + n for c, n in zip(self.counts, new)]
        need = [-(-c // self.page_size) - len(h) for c, h in zip(counts, self.held)]
        if sum(need) > len(self.free):
            raise RuntimeError(f"page pool exhausted: {sum(need)} more pages of {self.page_size} needed, {len(self.free)} free")
        self.counts = counts
        if not any(need):
            return
        for pages, n in zip(self.held, need):
            pages.extend(self.free.pop() for _ in range(n))
        blocks = max(len(h) for h in self.held)
        rows = [h + [-1] * (blocks - len(h)) for h in self.held]
        self.table = torch.tensor(rows, dtype=torch.int32, device=self.device)


def _text_model(model):
    inner = model.model
    return getattr(inner, "language_model", inner)


class PagedDecoder:
    """Runs a north_mini_code (Cohere2Moe) or deepseek_ocr_2 text model on a page pool of ``pages`` pages."""

    def __init__(self, model, pages: int, page_size: int = PAGE_SIZE):
        text = _text_model(model)
        kind = type(text).__name__
        if kind not in ("Cohere2MoeModel", "DeepseekOcr2TextModel"):
            raise RuntimeError(f"PagedDecoder runs Cohere2MoeModel and DeepseekOcr2TextModel, not {kind}")
        self.model, self.text, self.parallel = model, text, kind == "Cohere2MoeModel"
        cfg = text.config
        weight = text.embed_tokens.weight
        head_dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
        self.heads, self.kv_heads, self.dim = cfg.num_attention_heads, cfg.num_key_value_heads, head_dim
        self.inv_freq = text.rotary_emb.inv_freq.to(weight.device, torch.float32).contiguous()  # also of a model cast whole
        self.scale = float(getattr(text.rotary_emb, "attention_scaling", 1.0))
        self.logit_scale = float(getattr(cfg, "logit_scale", None) or 1.0) if self.parallel else 1.0
        self.pool = PagePool(len(text.layers), pages, self.kv_heads, head_dim, weight.dtype, weight.device, page_size)

    def _norm(self, norm, x):
        if not self.parallel:  # RMS norm: the model's own
            return norm(x)
        return ops.layer_norm(x, norm.weight, getattr(norm, "bias", None), norm.variance_epsilon)

    def _attention(self, i: int, attn, x, lengths, offsets, most: int):
        tokens = x.shape[0]
        q, k, v = (proj(x).view(tokens, -1, self.dim) for proj in (attn.q_proj, attn.k_proj, attn.v_proj))
        window = int(getattr(attn, "sliding_window", None) or 0)
        # Cohere2's layers without a window carry no positions, except where the model says so
        turned = not self.parallel or window > 0 or bool(getattr(attn, "force_rope", False))
        pool = self.pool
        out = ops.paged_append(k, v, pool.k[i], pool.v[i], pool.table, lengths, offsets, q=q if turned else None,
                               inv_freq=self.inv_freq if turned else None, interleaved=self.parallel, scale=self.scale)
        out = ops.paged_attention(out if turned else q, pool.k[i], pool.v[i], pool.table, lengths, offsets, scale=attn.scaling,
                                  window=window, max_new=most)
        return attn.o_proj(out.view(tokens, -1))

    def _mlp(self, mlp, x):
        y = mlp(x[None])
        return (y[0] if isinstance(y, tuple) else y)[0]

    @torch.no_grad()
    def step(self, tokens: list[torch.Tensor]) -> torch.Tensor:
        """Feeds tokens[b], the next tokens of sequence b (1-D, possibly none), to every open sequence; opens as many as there are if
        none is. Returns the logits behind each sequence's last new token [sequences, vocabulary] (of a sequence without new
        tokens: zeros)."""
        pool = self.pool
        if not pool.held:
            pool.open(len(tokens))
        if len(tokens) != len(pool.held):
            raise RuntimeError(f"{len(pool.held)} sequences are open, tokens for {len(tokens)} given")
        new = [int(t.numel()) for t in tokens]
        pool.grow(new)
        dev = pool.device
        ends = [0]
        for n in new:
            ends.append(ends[-1] + n)
        # one copy to the device: lengths and offsets
        both = torch.tensor(pool.counts + ends, dtype=torch.int32).to(dev)
        lengths, offsets = both[:len(new)], both[len(new):]
        if ends[-1] == 0:
            return torch.zeros(len(new), self.model.lm_head.out_features, device=dev, dtype=self.text.embed_tokens.weight.dtype)
        x = self.text.embed_tokens(torch.cat([t.reshape(-1).to(dev) for t in tokens]))
        most = max(new)
        for i, layer in enumerate(self.text.layers):
            h = self._norm(layer.input_layernorm, x)
            a = self._attention(i, layer.self_attn, h, lengths, offsets, most)
            if self.parallel:  # Cohere's block: attention and MLP read the same norm
                x = x + a + self._mlp(layer.mlp, h)
            else:
                x = x + a
                x = x + self._mlp(layer.mlp, layer.post_attention_layernorm(x))
        if ends[-1] != len(new) or any(n != 1 for n in new):
            x = x[[max(e - 1, 0) for e in ends[1:]]]
        logits = self.model.lm_head(self._norm(self.text.norm, x.contiguous())) * self.logit_scale
        idle = [b for b, n in enumerate(new) if n == 0]
        if idle:
            logits[idle] = 0
        return logits

    @torch.no_grad()
    def generate(self, prompts: list[torch.Tensor], n: int, chunk: int | None = None) -> torch.Tensor:
        """n greedy tokens behind each prompt [sequences, n]. ``chunk``: prompts enter in pieces of at most that many tokens."""
        self.pool.open(len(prompts))
        prompts = [p.reshape(-1) for p in prompts]
        longest = max(int(p.numel()) for p in prompts)
        size = longest if chunk is None else int(chunk)
        if n < 1 or size < 1 or min(int(p.numel()) for p in prompts) < 1:
            raise RuntimeError("prompts, chunks and continuations must hold at least one token")
        last = None
        for at in range(0, longest, size):
            logits = self.step([p[at:at + size] for p in prompts])
            fed = torch.tensor([at < p.numel() for p in prompts], device=logits.device)
            last = logits if last is None else torch.where(fed[:, None], logits, last)
        out = [last.argmax(-1)]
        while len(out) < n:
            out.append(self.step(list(out[-1].view(-1, 1).unbind())).argmax(-1))
        return torch.stack(out, 1)


def measure(model, inputs: dict, opts, reference) -> dict:
    """What modeling.main records of a variant, for the paged decoder on the model as it is: a prompt forward's median, the decode
    rate, and the greedy gate against ``reference``."""
    import time

    from cernels_amd.modeling import main as runner

    ids = inputs["input_ids"][0]
    longest = int(ids.numel()) + max(opts.gate_tokens, opts.decode_tokens) + 1
    decoder = PagedDecoder(model, pages=-(-longest // PAGE_SIZE))

    def prompt():
        decoder.pool.open(1)
        return decoder.step([ids])

    traced = runner.Trace(decoder.generate([ids], opts.gate_tokens)[0], prompt()[0].float())
    times, spent = [], 0.0
    while len(times) < 3 or spent < opts.prefill_seconds:
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        prompt()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e-3)
        spent += times[-1]
    prefill = statistics.median(times)
    best = float("inf")
    for _ in range(max(1, opts.decode_runs)):
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        decoder.generate([ids], opts.decode_tokens)
        torch.cuda.synchronize()
        best = min(best, time.perf_counter() - t0)
    rate = opts.decode_tokens / max(best - prefill, 1e-9)
    return {"prefill_ms": round(prefill * 1e3, 2), "decode_tok_s": round(rate, 2), "generate_s": round(best, 3),
            **traced.against(reference), "last_logits_std": round(float(reference.logits.std()), 4)}
