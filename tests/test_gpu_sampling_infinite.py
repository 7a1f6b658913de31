"""GPU: rows with infinite logits in every variant of the sampling kernel -- rows kept in shared memory or read again by each
pass, by one CTA or a cluster.  All weights are 0 or 1, so that borders are whole numbers and tokens exact."""
import math

import pytest
import torch

import qlinear
from test_gpu_sampling import BF, F32, HF, check, gen

pytestmark = pytest.mark.gpu

COUNTS = (1, 2, 3, 7, 100, 200, 400, 512, 513, 3000)


@pytest.mark.parametrize("rows,V,dtype", [
    (10, 5000, BF), (10, 128256, BF), (500, 5000, F32),  # in shared memory: a cluster, its longest slices, one CTA a row
    (120, 128256, BF), (60, 200001, F32), (10, 655104, HF),  # read again: clusters of 2, 4 and 16 CTAs
    (500, 128256, BF), (410, 70001, HF),  # .. one CTA
])
def test_infinite_logits_share_everything(rows, V, dtype):
    g = gen(V)
    few = len(COUNTS)
    x = (torch.randn(few, V, generator=g, device="cuda") * 2).to(dtype)
    for b, n in enumerate(COUNTS):
        x[b, torch.randperm(V, generator=g, device="cuda")[:n]] = -math.inf
        x[b, torch.randperm(V, generator=g, device="cuda")[:n]] = math.inf
    u = torch.rand(few, generator=g, device="cuda")
    times = -(-rows // few)
    many, numbers = x.repeat(times, 1), u.repeat(times)
    for s in (dict(), dict(top_p=0.9), dict(top_p=0.995), dict(top_p=0.999, temperature=0.7), dict(top_p=0.999, temperature=1.3, min_p=0.5),
              dict(top_p=0.997, temperature=0.35, top_k=2000), dict(top_k=5, top_p=0.999), dict(min_p=1.0), dict(temperature=0.0)):
        want = check(x, u, **s)
        assert int(want.min()) >= 0
        # what the outputs held before, were they not written
        junk = [torch.full((many.shape[0],), 1 << 40, device="cuda"), torch.full((many.shape[0],), 7.0, device="cuda")]
        del junk
        got, logprobs = qlinear.sample(many, numbers, logprobs=True, **{**dict(temperature=1.0), **s})
        assert torch.equal(got, want.repeat(times)), s
        assert torch.equal(logprobs, qlinear.sample(x, u, logprobs=True, **{**dict(temperature=1.0), **s})[1].repeat(times))
    assert qlinear.device_error() == 0
