"""CPU: what Decoder.generate does around its steps, with the passes themselves replaced."""
import pytest
import torch

from qlinear import cache as C
from qlinear import llama
from test_cache import small  # noqa: F401


class Passes:
    """A decoder whose pass takes a step of its Ahead and gives logits of 8 tokens; the `fails`-th raises."""

    def __init__(self, monkeypatch, fails=None, positions=1000):
        self.count, self.fails = 0, fails
        self.model = llama.Decoder.__new__(llama.Decoder)
        self.model.config = llama.Config(positions=positions, vocab=8)
        self.model.norm = torch.zeros(1)
        monkeypatch.setattr(C.Ahead, "next", lambda ahead: None)
        monkeypatch.setattr(llama.Decoder, "forward", self.forward)
        monkeypatch.setattr(llama.decoder, "sample", lambda x, u, **kw: x.argmax(-1))

    def forward(self, tokens, cache, step):
        self.count += 1
        if self.count == self.fails:
            raise MemoryError
        return torch.nn.functional.one_hot((tokens + 1) % 8, 8).to(torch.bfloat16)


@pytest.mark.parametrize("fails", [1, 2, 3, 5])
def test_a_step_that_fails_is_not_counted(small, monkeypatch, fails):  # noqa: F811
    p, c = Passes(monkeypatch, fails), small(20)
    seqs = [c.new(), c.new()]
    c.step(seqs, [15, 3])
    with pytest.raises(MemoryError):
        p.model.generate(c, seqs, torch.tensor([0, 4]), 5)
    assert [c.length(s) for s in seqs] == [15 + fails - 1, 3 + fails - 1]
    p.fails = None
    assert p.model.generate(c, seqs, torch.tensor([0, 4]), 3).tolist() == [[1, 2, 3], [5, 6, 7]]
    assert [c.length(s) for s in seqs] == [17 + fails, 5 + fails]


@pytest.mark.parametrize("new", [0, -1, -3])
def test_no_tokens(small, monkeypatch, new):  # noqa: F811
    p, c = Passes(monkeypatch), small(4)
    a = c.new()
    c.step([a], [5])
    out = p.model.generate(c, [a], torch.tensor([2]), new)
    assert out.shape == (1, 0) and out.dtype == torch.int64 and c.length(a) == 5 and p.count == 0


def test_a_vocabulary_past_the_rows_of_sampling(small, monkeypatch):  # noqa: F811
    """The most likely token needs no sampling; drawing one is refused as ever."""
    p, c = Passes(monkeypatch), small(4)
    logits = torch.zeros(1, llama.decoder.MAX_SAMPLE_ROW // 2 + 1, dtype=torch.bfloat16)
    logits[0, -1] = 1

    def sample(x, u, **kw):
        raise ValueError

    monkeypatch.setattr(llama.Decoder, "forward", lambda *a: logits)
    monkeypatch.setattr(llama.decoder, "sample", sample)
    a = c.new()
    c.step([a], [5])
    assert p.model.generate(c, [a], torch.tensor([2]), 2).tolist() == [[655104, 655104]]
    with pytest.raises(ValueError):
        p.model.generate(c, [a], torch.tensor([2]), 2, llama.Sampling())
    logits = logits[:, 1:]
    with pytest.raises(ValueError):
        p.model.generate(c, [a], torch.tensor([2]), 2)
    assert c.length(a) == 7
