"""GPU: the Llama-shaped decoder (quantized linears, norms, rotary append, paged attention, page
copies together) against a plain forward pass in 64 bits on the dequantized weights."""
import pytest
import torch

import qlinear
from qlinear.llama import Config, Decoder, main

pytestmark = pytest.mark.gpu

SMALL = Config(hidden=256, layers=2, heads=6, kv_heads=2, head_dim=64, ffn=512, vocab=1000, positions=4096)


def reference(model, tokens):
    """Logits of every position, [n, vocab], computed at once without a cache."""
    c = model.config
    w = lambda q: qlinear.dequantize(q.weight, q.scales, q.biases, c.group_size, c.bits).double()  # noqa: E731
    rms = lambda x, n: x / (x.square().mean(-1, keepdim=True) + c.eps).sqrt() * n.double()  # noqa: E731
    n = tokens.shape[0]
    cos, sin = (t.double()[:, None] for t in model.table[:n].chunk(2, 1))

    def turn(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    x = model.embedding(tokens).double()
    hide = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
    for ly in model.layers:
        q, k, v = (rms(x, ly.attn_norm) @ w(ly.qkv).T).view(n, -1, c.head_dim).split([c.heads, c.kv_heads, c.kv_heads], 1)
        q, k = turn(q), turn(k).repeat_interleave(c.heads // c.kv_heads, 1)
        v = v.repeat_interleave(c.heads // c.kv_heads, 1)
        p = torch.einsum("ihd,jhd->hij", q, k).div(c.head_dim ** 0.5).masked_fill(hide, -torch.inf).softmax(-1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ w(ly.out).T
        h = rms(x, ly.ffn_norm)
        x = x + (torch.nn.functional.silu(h @ w(ly.gate).T) * (h @ w(ly.up).T)) @ w(ly.down).T
    return rms(x, model.norm) @ w(model.head).T


def close(got, want):
    # bf16 activations: about 12 roundings (2^-8 relative, independent) on the way through a layer,
    # two layers; the logits' relative error is held to 2^-8 * sqrt(24) * 2
    assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -8 * 24 ** 0.5 * 2


def test_chunks_steps_forks_and_compaction_give_the_same_logits():
    model = Decoder.random(SMALL, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    tokens = torch.randint(0, SMALL.vocab, (230,), generator=g, device="cuda")
    want = reference(model, tokens)
    cache = model.cache(pages=60)
    other = cache.new()  # a neighbour in the pool, so that pages are not in order
    model.prompt(cache, other, tokens[:50])
    seq = cache.new()
    close(model.prompt(cache, seq, tokens[:200], chunk=77), want[199:200])       # chunks of a prompt
    for i in range(200, 205):                                                    # single tokens
        close(model.forward(tokens[i:i + 1], cache, cache.step([seq], [1])), want[i:i + 1])
    fork = cache.fork(seq)
    # a batch of single tokens and a chunk: the fork takes another token, the original goes on
    strange = torch.tensor([7], device="cuda")
    both = model.forward(torch.cat([strange, tokens[205:225]]), cache, cache.step([fork, seq], [1, 20]))
    close(both[1:], want[224:225])
    close(both[:1], reference(model, torch.cat([tokens[:205], strange]))[-1:])
    cache.free(other)
    a = model.forward(tokens[225:226], cache, cache.step([seq], [1]))
    cache.truncate(seq, 225)
    assert cache.compact() > 0
    b = model.forward(tokens[225:226], cache, cache.step([seq], [1]))
    assert torch.equal(a, b)  # moved pages, same arithmetic
    close(b, want[225:226])
    assert qlinear.device_error() == 0


def test_command_runs(capsys):
    main(["--layers", "1", "--prompt", "100", "--new", "8", "--forks", "3"])
    out = capsys.readouterr().out
    assert "ms a step" in out and "moved by compaction" in out
    assert qlinear.device_error() == 0
