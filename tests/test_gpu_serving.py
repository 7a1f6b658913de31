"""GPU: sampling, step planning and windows with sinks together, as the decoder runs them."""
import random

import pytest
import torch

import qlinear
from qlinear.cache import PagedCache
from qlinear.llama import Config, Decoder, Sampling, main
from test_gpu_llama import SMALL, close, reference

pytestmark = pytest.mark.gpu


def same(a, b):
    assert a.max_q == b.max_q and a.max_kv == b.max_kv and a.new_tokens == b.new_tokens and a.lengths == b.lengths
    for k in ("positions", "slots", "page_table", "q_starts", "kv_lens"):
        x, y = getattr(a, k), getattr(b, k)
        assert x.dtype == y.dtype and x.shape == y.shape and x.tolist() == y.tolist(), k


@pytest.mark.parametrize("seed", range(4))
def test_steps_on_the_gpu_are_those_of_the_books(seed):
    rng = random.Random(seed)
    caches = [PagedCache(1, 1, 16, 90, 16, device=d) for d in ("cuda", "cpu")]
    seqs = []
    for _ in range(60):
        op = rng.choice(["new", "step", "step", "step", "truncate", "evict"])
        if op == "new" or not seqs:
            seqs.append([c.new() for c in caches][0])
        elif op == "step":
            pick = rng.sample(seqs, rng.randint(1, len(seqs)))
            n = [rng.choice([0, 1, 1, 7, 40]) for _ in pick]
            if not sum(n):
                continue
            try:
                a, b = (c.step(pick, n) for c in caches)
            except qlinear.OutOfPages:
                q = seqs.pop(0)
                for c in caches:
                    c.free(q)
                continue
            same(a, b)
        else:
            q = rng.choice(seqs)
            for c in caches:
                if op == "evict":
                    c.evict(q, 20, 5)
                elif q not in c._least:
                    c.truncate(q, c.length(q) // 2)
    assert qlinear.device_error() == 0


@pytest.mark.parametrize("graph", [False, True])
def test_steps_planned_ahead(graph):
    """The tensors of each step are those that the cache would have made."""
    caches = [PagedCache(1, 1, 16, 40, 16) for _ in range(2)]
    for c in caches:
        seqs = [c.new() for _ in range(3)]
        c.step(seqs, [3, 16, 30])
        seqs.append(c.fork(seqs[2]))
    steps = 37
    ahead = caches[0].ahead(seqs, steps)
    got = ahead.next()
    if graph:
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            ahead.next()
    slots = []
    for i in range(steps):
        if i:
            captured.replay() if graph else ahead.next()
        want = caches[1].step(seqs, [1] * 4)
        assert got.positions.tolist() == want.positions.tolist() and got.q_starts.tolist() == want.q_starts.tolist()
        assert got.kv_lens.tolist() == want.kv_lens.tolist() and got.max_q == 1 and got.max_kv == 30 + steps
        table = got.page_table.tolist()
        assert got.slots.tolist() == [table[b][p // 16] * 16 + p % 16 for b, p in enumerate(want.positions.tolist())]
        slots += got.slots.tolist()
    assert len(set(slots)) == len(slots)  # no place twice
    ahead.close(steps)
    for b, s in enumerate(seqs):
        assert caches[0].pages_of(s) == table[b][:len(caches[0].pages_of(s))]
    got = ahead.next()  # one step too many finds no room, here as its sequences end a page
    torch.cuda.synchronize()
    assert caches[0].free_pages == caches[1].free_pages
    assert qlinear.device_error() in (0, qlinear._lib.DEV_ERR_NO_ROOM)


def old_generate(model, cache, seqs, tokens, new):
    """Step by step from the cache's books."""
    out = []
    for _ in range(new):
        tokens = model.forward(tokens, cache, cache.step(seqs, [1] * len(seqs))).argmax(-1)
        out.append(tokens)
    return torch.stack(out, 1)


@pytest.mark.parametrize("graph", [False, True])
def test_greedy_continuations(graph):
    model = Decoder.random(SMALL, seed=5)
    tokens = torch.randint(0, SMALL.vocab, (90,), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    first = torch.tensor([3, 5, 7], device="cuda")
    texts, logits = [], []
    for way in (lambda *a: old_generate(model, *a), lambda *a: model.generate(*a, graph=graph)):
        cache = model.cache(pages=60)
        seq = cache.new()
        model.prompt(cache, seq, tokens)
        seqs = [seq, cache.fork(seq), cache.fork(seq)]
        texts.append(way(cache, seqs, first, 40))
        logits.append(model.forward(first, cache, cache.step(seqs, [1] * 3)))
        assert [cache.length(s) for s in seqs] == [131] * 3
    assert torch.equal(*texts) and torch.equal(*logits)
    assert qlinear.device_error() == 0


@pytest.mark.parametrize("settings", [dict(temperature=0.8, top_p=0.9), dict(top_k=20), dict(temperature=1.5, min_p=0.02)], ids=str)
def test_sampled_continuations(settings):
    """Given random numbers give the same text, replayed or not, alone or in a batch; every token is the one
    that the step's logits and its number give."""
    model = Decoder.random(SMALL, seed=7)
    g = torch.Generator(device="cuda").manual_seed(8)
    tokens = torch.randint(0, SMALL.vocab, (50,), generator=g, device="cuda")
    first, u = torch.tensor([3, 5], device="cuda"), torch.rand((30, 2), generator=g, device="cuda")
    texts = []
    for graph in (False, True):
        cache = model.cache(pages=40)
        seq = cache.new()
        model.prompt(cache, seq, tokens)
        texts.append(model.generate(cache, [seq, cache.fork(seq)], first, 30, Sampling(**settings), u, graph))
    assert torch.equal(*texts) and texts[0].shape == (2, 30)
    cache = model.cache(pages=40)
    seq = cache.new()
    model.prompt(cache, seq, tokens)
    seqs = [seq, cache.fork(seq)]
    current = first
    for i in range(30):
        current = qlinear.sample(model.forward(current, cache, cache.step(seqs, [1, 1])), u[i], **settings)
        assert torch.equal(current, texts[0][:, i])
    # numbers of its own
    more = model.generate(cache, seqs, current, 5, Sampling(**settings))
    assert more.shape == (2, 5) and int(more.min()) >= 0 and int(more.max()) < SMALL.vocab
    with pytest.raises(ValueError):
        model.generate(cache, seqs, current, 5, Sampling(**settings), u)
    assert [cache.length(s) for s in seqs] == [85, 85]
    assert qlinear.device_error() == 0


def test_window_with_sinks_in_the_decoder(monkeypatch):
    """Chunks of a prompt, single tokens, steps ahead and evicted pages against a plain forward pass with the window's mask."""
    config = Config(**{**SMALL.__dict__, "window": 40, "sinks": 5})
    model = Decoder.random(config, seed=9)
    g = torch.Generator(device="cuda").manual_seed(10)
    tokens = torch.randint(0, SMALL.vocab, (260,), generator=g, device="cuda")
    i, j = torch.arange(260, device="cuda")[:, None], torch.arange(260, device="cuda")
    with monkeypatch.context() as m:  # the reference's mask
        m.setattr(torch.Tensor, "triu", lambda self, k=0: (j > i) | ((j <= i - 40) & (j >= 5)))
        want = reference(model, tokens)
    cache = model.cache(pages=12)  # 192 positions: not enough without eviction
    seq = cache.new()
    close(model.prompt(cache, seq, tokens[:200], chunk=61), want[199:200])
    assert cache.pages - cache.free_pages <= 5 and cache.pages_of(seq)[1] == -1
    for n in range(200, 210):
        close(model.forward(tokens[n:n + 1], cache, cache.step([seq], [1])), want[n:n + 1])
    close(model.forward(tokens[210:240], cache, cache.step([seq], [30])), want[239:240])
    cache.evict(seq, 40, 5)
    text = model.generate(cache, [seq], tokens[240:241], 10, graph=True)
    # (the first token of the continuation; the reference does not know the others)
    if float(want[240].topk(2).values.diff().abs()) > 0.2:
        assert int(text[0, 0]) == int(want[240].argmax())
    assert cache.length(seq) == 250 and cache.pages - cache.free_pages <= 5
    assert qlinear.device_error() == 0


def test_command_samples_in_a_window(capsys):
    main(["--layers", "1", "--prompt", "100", "--new", "20", "--forks", "3", "--temperature", "0.8", "--top-p", "0.9", "--top-k", "50",
          "--window", "64", "--sinks", "4", "--graph"])
    assert "ms a step" in capsys.readouterr().out
    assert qlinear.device_error() == 0
