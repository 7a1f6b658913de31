"""A Llama-shaped decoder on the quantized linears and the decoder operators: the prompt-refine
path (Llama-3.2-3B: hidden 3072, 28 layers, 24 query and 8 key / value heads of 128, SwiGLU 8192) with
chunked prompts, batched decoding, and continuations that share their prompt's pages.

    python -m qlinear.llama --layers 28 --prompt 700 --new 64 --forks 4

runs it on random weights (no checkpoint is read here; ``qlinear.io`` loads packed ones) and prints
the prompt's and the decode step's times.
"""
from __future__ import annotations

import argparse
from dataclasses import dataclass, field
from typing import List, Optional, Sequence

import torch

from . import decoder, ops
from .cache import PagedCache, Step
from .nn import Linear, QuantizedLinear, TokenEmbedding


@dataclass
class Config:
    """Llama-3.2-3B's sizes and rotary scaling (None: plain frequencies)."""

    hidden: int = 3072
    layers: int = 28
    heads: int = 24
    kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 8192
    vocab: int = 128256
    positions: int = 131072
    rope_base: float = 500000.0
    rope_scaling: Optional[dict] = field(default_factory=lambda: {
        "type": "llama3", "factor": 32.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_positions": 8192})
    eps: float = 1e-5
    bits: int = 4
    group_size: int = 64


@dataclass
class Layer:
    attn_norm: torch.Tensor
    qkv: QuantizedLinear
    out: QuantizedLinear
    ffn_norm: torch.Tensor
    gate: QuantizedLinear
    up: QuantizedLinear
    down: QuantizedLinear


class Decoder:
    def __init__(self, config: Config, embedding: TokenEmbedding, layers: List[Layer], norm: torch.Tensor, head: QuantizedLinear):
        self.config, self.embedding, self.layers, self.norm, self.head = config, embedding, layers, norm, head
        self.table = decoder.rope_table(config.head_dim, config.positions, config.rope_base, config.rope_scaling, device=norm.device)

    @staticmethod
    def random(config: Config, seed: int = 0, device="cuda") -> "Decoder":
        g = torch.Generator(device=device).manual_seed(seed)
        c = config

        def lin(n, k):
            w = (torch.randn(n, k, generator=g, device=device) * k ** -0.5).to(torch.bfloat16)
            return QuantizedLinear.try_from_linear(Linear(w), c.group_size, c.bits)

        def norm():
            return (1 + 0.1 * torch.randn(c.hidden, generator=g, device=device)).to(torch.bfloat16)

        layers = [Layer(norm(), lin((c.heads + 2 * c.kv_heads) * c.head_dim, c.hidden), lin(c.hidden, c.heads * c.head_dim), norm(),
                        lin(c.ffn, c.hidden), lin(c.ffn, c.hidden), lin(c.hidden, c.ffn)) for _ in range(c.layers)]
        table = TokenEmbedding(torch.randn(c.vocab, c.hidden, generator=g, device=device).to(torch.bfloat16))
        table.quantize(c.bits, True)
        return Decoder(c, table, layers, norm(), lin(c.vocab, c.hidden))

    def cache(self, pages: int, page_size: int = 16) -> PagedCache:
        c = self.config
        return PagedCache(c.layers, c.kv_heads, c.head_dim, pages, page_size, device=self.norm.device)

    def forward(self, tokens: torch.Tensor, cache: PagedCache, step: Step) -> torch.Tensor:
        """Logits of each sequence's last new token, [B, vocab]; the cache gets the new tokens.  Every
        sequence of the step needs one at least, and none may pass the table's positions (ValueError;
        the cache counts the step's tokens all the same, until they are truncated)."""
        c = self.config
        if step.new_tokens is not None and min(step.new_tokens) == 0:
            raise ValueError(f"a step with sequences without new tokens {step.new_tokens} has no logits for them")
        if step.lengths is not None:
            self._fits(max(step.lengths))
        x = self.embedding(tokens).to(torch.bfloat16)
        T = x.shape[0]
        h, x = decoder.norm_residual(x, torch.zeros_like(x), self.layers[0].attn_norm, eps=c.eps)
        for i, ly in enumerate(self.layers):
            qkv = ly.qkv.forward(h).view(T, c.heads + 2 * c.kv_heads, c.head_dim)
            q, k, v = qkv.split([c.heads, c.kv_heads, c.kv_heads], 1)
            kc, vc = cache.layer(i)
            q = decoder.rope_append(q, k, v, self.table, step.positions, kc, vc, step.slots)
            a = decoder.paged_attention(q, kc, vc, step.page_table, step.q_starts, step.kv_lens, max_q=step.max_q, max_kv=step.max_kv)
            h, x = decoder.norm_residual(ly.out.forward(a.view(T, -1)), x, ly.ffn_norm, eps=c.eps)
            f = ops.quantized_matmul(h, ly.gate.weight, ly.gate.scales, ly.gate.biases, True, c.group_size, c.bits, act="swiglu",
                                     up=(ly.up.weight, ly.up.scales, ly.up.biases))
            following = self.layers[i + 1].attn_norm if i + 1 < len(self.layers) else self.norm
            h, x = decoder.norm_residual(ly.down.forward(f), x, following, eps=c.eps)
        last = (step.q_starts[1:] - 1).long()
        return self.head.forward(h[last])

    def _fits(self, length: int) -> None:
        """The rotary table's end is known here; past it the kernels would give zeros and report it."""
        if length > self.config.positions:
            raise ValueError(f"a sequence of {length} tokens: the decoder's table holds {self.config.positions} positions")

    def generate(self, cache: PagedCache, seqs: Sequence[int], tokens: torch.Tensor, new: int) -> torch.Tensor:
        """Greedy continuation of sequences from their next tokens [B]: [B, new] token ids."""
        self._fits(max(cache.length(s) for s in seqs) + new)
        out = []
        for _ in range(new):
            logits = self.forward(tokens, cache, cache.step(seqs, [1] * len(seqs)))
            tokens = logits.argmax(-1)
            out.append(tokens)
        return torch.stack(out, 1) if out else tokens.new_empty((len(seqs), 0))

    def prompt(self, cache: PagedCache, seq: int, tokens: torch.Tensor, chunk: int = 2048) -> torch.Tensor:
        """Appends a prompt [n] in chunks; returns the last token's logits [1, vocab]."""
        if tokens.shape[0] < 1 or chunk < 1:
            raise ValueError(f"a prompt needs at least one token and a chunk of one (got {tokens.shape[0]} tokens, chunk {chunk})")
        self._fits(cache.length(seq) + tokens.shape[0])
        for at in range(0, tokens.shape[0], chunk):
            part = tokens[at:at + chunk]
            logits = self.forward(part, cache, cache.step([seq], [part.shape[0]]))
        return logits


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description="Llama-shaped decoder on random weights")
    ap.add_argument("--layers", type=int, default=28)
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--chunk", type=int, default=2048)
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--forks", type=int, default=4, help="continuations that share the prompt's pages")
    a = ap.parse_args(argv)
    model = Decoder.random(Config(layers=a.layers))
    per = -(-(a.prompt + a.new) // 16) + 1
    cache = model.cache(pages=per + a.forks * (a.new // 16 + 2))
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, model.config.vocab, (a.prompt,), generator=g, device="cuda")
    warm = cache.new()
    model.prompt(cache, warm, tokens, a.chunk)
    cache.free(warm)
    marks = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
    seq = cache.new()
    marks[0].record()
    logits = model.prompt(cache, seq, tokens, a.chunk)
    marks[1].record()
    seqs = [seq] + [cache.fork(seq) for _ in range(a.forks - 1)]
    first = logits.topk(len(seqs)).indices[0]  # each continuation starts from another token
    text = model.generate(cache, seqs, first, a.new)
    marks[2].record()
    torch.cuda.synchronize()
    print(f"prompt of {a.prompt} tokens: {marks[0].elapsed_time(marks[1]):.2f} ms; {a.new} tokens for {len(seqs)} continuations: "
          f"{marks[1].elapsed_time(marks[2]) / max(a.new, 1):.3f} ms a step; pages in use {cache.pages - cache.free_pages} of {cache.pages}")
    for s in seqs[1:]:
        cache.free(s)
    moved = cache.compact()
    print(f"after freeing the forks: {cache.pages - cache.free_pages} pages in use, {moved} moved by compaction; first ids {text[0, :8].tolist()}")


if __name__ == "__main__":
    main()
