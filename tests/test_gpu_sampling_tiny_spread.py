"""GPU: logits that differ by next to nothing, or by all that the type holds: the order stays, whatever the weights."""
import pytest
import torch

import qlinear
from test_gpu_sampling import BF, F32, check, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [600, 5000, 128256])
@pytest.mark.parametrize("top_k", [1, 7, 50, 300, 512, 2000])
@pytest.mark.parametrize("unit", [2.0 ** -149, 2.0 ** -140, 2.0 ** -133])
def test_logits_next_to_zero(V, top_k, unit):
    """Distinct logits within 2^-116 of 0 (subnormal ones among them): every weight is 1 and the first k of the order stay."""
    g = gen(V + top_k)
    x = (torch.stack([torch.randperm(V, generator=g, device="cuda") for _ in range(4)]) - V // 3).double().mul(unit).float()
    u = torch.rand(4, generator=g, device="cuda")
    for s in (dict(), dict(top_p=0.5), dict(top_p=0.9999999), dict(min_p=1.0)):
        token = check(x, u, top_k=top_k, **s)
        if not s and top_k < V:  # the drawn one of the k largest, by index
            order = x.sort(descending=True, stable=True).indices[:, :top_k].sort().values
            assert torch.equal(token, order.gather(1, (u.double() * top_k).long()[:, None])[:, 0])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_logits_over_all_that_the_type_holds(dtype):
    g = gen(9)
    x = ((torch.rand(4, 5000, generator=g, device="cuda") * 2 - 1) * torch.finfo(dtype).max).to(dtype).clamp(torch.finfo(dtype).min, torch.finfo(dtype).max)
    x[:, 17], x[:, 18] = torch.finfo(dtype).max, torch.finfo(dtype).min
    for s in (dict(top_k=7), dict(top_k=600), dict(top_k=40, top_p=0.5), dict(top_p=0.9)):
        check(x, torch.rand(4, generator=g, device="cuda"), **s)
    assert qlinear.device_error() == 0
