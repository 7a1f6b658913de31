"""CPU: what the Llama-shaped decoder refuses on the host, before anything is launched."""
import pytest
import torch

from qlinear.cache import PagedCache
from qlinear.llama import Config, Decoder

TINY = Config(hidden=64, layers=1, heads=1, kv_heads=1, head_dim=64, ffn=64, vocab=10, positions=40)


@pytest.fixture
def model():
    return Decoder(TINY, None, [], torch.ones(64), None)


def cache():
    return PagedCache(1, 1, 64, 8, device="cpu")


@pytest.mark.parametrize("counts", [[0, 3], [3, 0], [1, 0, 1]])
def test_forward_refuses_sequences_without_new_tokens(model, counts):
    """Their logits would be another sequence's."""
    c = cache()
    step = c.step([c.new() for _ in counts], counts)
    with pytest.raises(ValueError, match="without new tokens"):
        model.forward(torch.zeros(sum(counts), dtype=torch.int64), c, step)


def test_positions_past_the_table_are_refused(model):
    c = cache()
    a = c.new()
    step = c.step([a], [41])
    with pytest.raises(ValueError, match="40 positions"):
        model.forward(torch.zeros(41, dtype=torch.int64), c, step)
    c.truncate(a, 38)
    with pytest.raises(ValueError, match="40 positions"):
        model.prompt(c, a, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="40 positions"):
        model.generate(c, [a], torch.zeros(1, dtype=torch.int64), 3)
    assert c.length(a) == 38 and c.free_pages == 5  # refused before the cache changed


def test_empty_prompts_and_continuations(model):
    c = cache()
    a = c.new()
    with pytest.raises(ValueError, match="at least one token"):
        model.prompt(c, a, torch.zeros(0, dtype=torch.int64))
    with pytest.raises(ValueError, match="chunk"):
        model.prompt(c, a, torch.zeros(3, dtype=torch.int64), chunk=0)
    assert model.generate(c, [a], torch.zeros(1, dtype=torch.int64), 0).shape == (1, 0)


def test_default_table_has_the_models_scaling():
    """Llama-3.2-3B stretches a context of 8192: wavelengths above 8192 by 32, below 2048 not at all,
    a linear blend (in turns) between."""
    n, c = 64, Config()
    f = c.rope_base ** (-torch.arange(n, dtype=torch.float64) / n)
    turns = 8192 * f / (2 * torch.pi)
    keep = ((turns - 1) / 3).clamp(0, 1)
    a = (f * keep + f / 32 * (1 - keep)) * 1000
    table = Decoder(Config(layers=0, positions=1001), None, [], torch.ones(1), None).table[1000].double()
    # the angle in fp64, its cosine and sine rounded to fp32
    assert float((table - torch.cat([a.cos(), a.sin()])).abs().max()) < 1e-6
