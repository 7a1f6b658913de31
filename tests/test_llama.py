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
