"""GPU: continuations in a window with sinks -- pages given back, steps planned ahead, replayed -- give the tokens and logits of
single steps from the cache's books that give nothing back."""
import pytest
import torch

import qlinear
from qlinear.llama import Config, Decoder, Sampling
from test_gpu_llama import SMALL

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("window,sinks", [(40, 5), (16, 33), (300, 17)])  # (the last is divided among CTAs)
@pytest.mark.parametrize("settings", [None, dict(temperature=0.9, top_p=0.9)], ids=str)
def test_window_continuations(monkeypatch, window, sinks, graph, settings):
    """The same division of the work on both sides (windows shorter than every length), so the same bits."""
    model = Decoder.random(Config(**{**SMALL.__dict__, "window": window, "sinks": sinks}), seed=11)
    g = torch.Generator(device="cuda").manual_seed(12)
    tokens = torch.randint(0, SMALL.vocab, (403,), generator=g, device="cuda")
    first, u = torch.tensor([3, 5], device="cuda"), torch.rand((45, 2), generator=g, device="cuda")
    texts, logits, used = [], [], []
    for evicting in (False, True):
        with monkeypatch.context() as m:
            if not evicting:
                m.setattr(Decoder, "_evict", lambda *a: None)
            cache = model.cache(pages=80)
            seq = cache.new()
            model.prompt(cache, seq, tokens, chunk=150)
            seqs = [seq, cache.fork(seq)]
            if evicting:
                texts.append(model.generate(cache, seqs, first, 45, Sampling(**settings) if settings else None, u if settings else None, graph))
            else:
                current, text = first, []
                for i in range(45):  # over three ends of pages
                    x = model.forward(current, cache, cache.step(seqs, [1, 1]))
                    current = qlinear.sample(x, u[i], **settings) if settings else x.argmax(-1)
                    text.append(current)
                texts.append(torch.stack(text, 1))
            used.append(cache.pages - cache.free_pages)
            logits.append(model.forward(texts[-1][:, -1].contiguous(), cache, cache.step(seqs, [1, 1])))
            assert [cache.length(s) for s in seqs] == [449, 449]
    assert torch.equal(*texts) and torch.equal(*logits)
    assert used[1] < used[0]
    assert qlinear.device_error() == 0
