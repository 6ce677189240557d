"""Beam search on the device: the choice of the beams, their history, and a Qwen3 decoder driven by it.

A step runs without the host looking at anything: logits of all beams -> `ops.beam_select` -> page reordering of the
beams' own caches -> the next token through the layers, whose attention reads the prompt's cache once for all beams
(`paged.shared_prefix_attention`).  The reference decodes one continuation per sequence."""
from __future__ import annotations

import torch

from . import ops
from .decoder import KvCache, Qwen3Decoder
from .paged import DEFAULT_KV_PAGE_SIZE, PagedKvCache, PagedLayers, shared_prefix_attention


class BeamSearch:
    """The `beams` best continuations of each of `groups` sequences.  Every `step` takes the logits of all beams
    ([groups * beams, vocab], beam b of group g in row g * beams + b) and leaves the choice in `parents` / `tokens` of that
    step; scores and end marks are updated in place, best beam first."""

    def __init__(self, groups: int, beams: int, max_steps: int, device, eos: int = -1):
        if groups < 1 or not 1 <= beams <= 32 or max_steps < 1:
            raise ValueError("BeamSearch: at least one group and step, 1 to 32 beams")
        self.groups, self.beams, self.max_steps, self.eos = groups, beams, max_steps, eos
        self.scores = torch.full((groups, beams), float("-inf"), device=device, dtype=torch.float32)
        self.scores[:, 0] = 0.0                       # one live beam until the first choice
        self.finished = torch.zeros(groups, beams, device=device, dtype=torch.uint8) if eos >= 0 else None
        self.parents = torch.zeros(max_steps, groups, beams, device=device, dtype=torch.int32)
        self.tokens = torch.zeros(max_steps, groups, beams, device=device, dtype=torch.int32)
        self.steps = 0

    def step(self, logits: torch.Tensor):
        """Chooses the next beams; returns (parents, tokens) [groups, beams] of this step."""
        if self.steps >= self.max_steps:
            raise ValueError(f"BeamSearch: {self.max_steps} steps have been taken")
        parents, tokens = self.parents[self.steps], self.tokens[self.steps]
        ops.beam_select(logits, self.scores, finished=self.finished, eos=self.eos, out=(self.scores, parents, tokens, self.finished))
        self.steps += 1
        return parents, tokens

    def all_finished(self) -> bool:
        """Whether every beam has ended (reads the marks back from the device)."""
        return self.finished is not None and bool(self.finished.all())

    def sequences(self, n_best: int = 1, length_penalty: float = 0.0):
        """The n_best token sequences of every group, [groups, n_best, steps] int32 (a finished one goes on with eos), and
        their scores: log-probability / length ** length_penalty, length counting the tokens up to the first eos."""
        if not 1 <= n_best <= self.beams:
            raise ValueError(f"sequences: 1 to {self.beams} of the beams")
        dev = self.scores.device
        order = torch.arange(self.beams, device=dev, dtype=torch.int32).expand(self.groups, -1).contiguous()
        if length_penalty == 0.0:                     # the beams are in order of score
            order = order[:, :n_best].contiguous()
            return ops.beam_trace(self.parents[:self.steps], self.tokens[:self.steps], order), self.scores[:, :n_best].clone()
        paths = ops.beam_trace(self.parents[:self.steps], self.tokens[:self.steps], order)
        ended = (paths == self.eos).cumsum(-1) > 0 if self.eos >= 0 else torch.zeros_like(paths, dtype=torch.bool)
        length = (~ended).sum(-1) + ended.any(-1)     # the first eos counts
        scores = self.scores / length.clamp(min=1).to(torch.float32) ** length_penalty
        best = torch.sort(scores, dim=-1, descending=True, stable=True).indices[:, :n_best]
        return torch.gather(paths, 1, best[..., None].expand(-1, -1, paths.shape[-1])), torch.gather(scores, 1, best)


class Qwen3BeamDecoder:
    """Beam search over a Qwen3 decoder from prompts of one length whose keys and values are in dense caches.  The prompt of each sequence
    is stored once per layer in pages (`quantization`); the beams add tokens to pages of their own (`own_quantization`)."""

    def __init__(self, decoder: Qwen3Decoder, caches: list[KvCache], prompt_len: int, beams: int, max_new_tokens: int, eos: int = -1,
                 quantization: str = "none", own_quantization: str = "none", page_size: int = DEFAULT_KV_PAGE_SIZE):
        if len(caches) != len(decoder.layers):
            raise ValueError("Qwen3BeamDecoder: one cache per layer")
        if prompt_len < 1 or prompt_len > caches[0].capacity:
            raise ValueError("Qwen3BeamDecoder: the caches hold no such prompt")
        self.decoder, self.prompt_len, self.beams = decoder, prompt_len, beams
        groups, kvh, _, d = caches[0].k.shape
        dev = caches[0].k.device
        self.prefixes = []
        for c in caches:
            prefix = PagedKvCache(groups, kvh, d, prompt_len, dev, quantization, page_size)
            prefix.append(c.k[:, :, :prompt_len].transpose(1, 2).contiguous(), c.v[:, :, :prompt_len].transpose(1, 2).contiguous())
            self.prefixes.append(prefix)
        self.own = PagedLayers.allocate(len(caches), groups * beams, kvh, d, max_new_tokens, dev, own_quantization, page_size)
        self.search = BeamSearch(groups, beams, max_new_tokens, dev, eos)
        self.held = 0                                  # tokens each beam has cached

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        """One token of every beam, [groups * beams] int32, through the layers: logits [groups * beams, vocab] fp32."""
        if self.held >= self.search.max_steps:
            raise ValueError(f"forward: the beams hold {self.held} tokens, all they were given room for")
        dec, w = self.decoder, self.decoder.w
        b, pos = tokens.numel(), self.prompt_len + self.held
        cos_half, sin_half = dec.rope_tables(pos, b)
        qd, kd = w.heads * w.head_dim, w.kv_heads * w.head_dim
        out, stream = ops.embed_rows(dec.embed, tokens.reshape(-1)), None
        for layer, prefix, own in zip(dec.layers, self.prefixes, self.own.caches):
            lw = layer.w
            if stream is None:
                x, normed = out, ops.rms_norm(out, lw.input_layernorm, lw.eps)
            else:
                normed, x = ops.rms_norm(out, lw.input_layernorm, lw.eps, residual=stream, return_sum=True)
            qkv = ops.linear(normed, lw.qkv, lw.fmt, n=qd + 2 * kd, k=lw.hidden)
            q = qkv[:, :qd].reshape(b, lw.heads, lw.head_dim)
            k = qkv[:, qd:qd + kd].reshape(b, lw.kv_heads, lw.head_dim)
            v = qkv[:, qd + kd:].reshape(b, 1, lw.kv_heads, lw.head_dim).contiguous()
            if lw.q_norm is not None:
                q, k = ops.rms_norm(q, lw.q_norm, lw.eps), ops.rms_norm(k, lw.k_norm, lw.eps)
            else:
                q, k = q.contiguous(), k.contiguous()
            ops.rope_pair_(q, k, cos_half, sin_half)
            own.append(k.reshape(b, 1, lw.kv_heads, lw.head_dim), v)
            attn = shared_prefix_attention(q, prefix, own, max_seq_len=self.held + 1)
            o = ops.linear(attn.reshape(b, qd), lw.o, lw.fmt, n=lw.hidden, k=qd)
            normed, stream = ops.rms_norm(o, lw.post_attention_layernorm, lw.eps, residual=x, return_sum=True)
            gu = ops.linear(normed, lw.gate_up, lw.fmt, n=2 * lw.intermediate, k=lw.hidden)
            act = ops.silu_mul(gu[:, :lw.intermediate], gu[:, lw.intermediate:])
            out = ops.linear(act, lw.down, lw.fmt, n=lw.hidden, k=lw.intermediate)
        self.held += 1
        hidden = ops.rms_norm(out, dec.final_norm, w.eps, residual=stream)
        return ops.linear(hidden, dec.lm_head, dec.lm_head_fmt, n=dec.embed.shape[0], k=w.hidden, out_dtype=torch.float32)

    def choose(self, logits: torch.Tensor) -> torch.Tensor:
        """The next beams from the logits of all beams: their tokens [groups * beams]; the caches follow the choice."""
        parents, tokens = self.search.step(logits)
        if self.held:
            self.own.use(self.own.reorder(parents))
        return tokens.reshape(-1)

    def generate(self, prompt_logits: torch.Tensor, n_best: int = 1, length_penalty: float = 0.0):
        """prompt_logits [groups, vocab]: what the prompt's last token gave.  Runs until max_new_tokens; returns
        `BeamSearch.sequences`."""
        tokens = self.choose(prompt_logits.repeat_interleave(self.beams, dim=0))
        while self.search.steps < self.search.max_steps:
            tokens = self.choose(self.forward(tokens))
        return self.search.sequences(n_best, length_penalty)
