"""GPU: sampling against its definition in 64 bits.

Tokens are whole numbers and must be equal.  The weights are whole multiples of 2^-S (S = 46, for more than 2^17
tokens 63 - ceil(log2 V)), so a border lies within V * 2^-(S + 1) of the definition's, relative to a sum of at
least 1, and that of float64 sums within V * 2^-53: below 2^-29 for random rows, whose u has 24 bits and hits such a
neighbourhood with a chance under 2^-29 for each token that stays.  Rows made of equal weights have borders that both
sides represent exactly."""
import math

import pytest
import torch

import qlinear

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
PLAIN = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def definition(x, u, temperature, top_k, top_p, min_p):
    """(token, log-probability) of one row."""
    x = x.double()
    if bool(x.isnan().any()) or float(x.max()) == -math.inf or any(map(math.isnan, (u, temperature, top_p, min_p))) or temperature < 0:
        return -1, math.nan
    order = torch.sort(x, descending=True, stable=True).indices
    if temperature == 0:
        return int(order[0]), 0.0
    top = x.max()
    d = torch.where(x == top, 0.0, x - top)[order]  # inf - inf is 0 here
    w = torch.exp(d / temperature)
    w = torch.where(d == -math.inf, 0.0, w)  # (an infinite temperature)
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        sums = w.cumsum(0)
        w = w[:1 + int((sums < top_p * sums[-1]).sum())]
    w = w[:max(1, int((w >= min_p).sum()))]
    index, back = torch.sort(order[:w.shape[0]])
    w = w[back]
    sums = w.cumsum(0)
    at = int((sums <= max(u, 0.0) * sums[-1]).sum())
    if at >= w.shape[0]:
        at = int(torch.nonzero(w)[-1])
    return int(index[at]), math.log(float(w[at]) / float(sums[-1]))


def check(x, u, **kw):
    kw = {**PLAIN, **kw}
    tokens, logprobs = qlinear.sample(x, u, logprobs=True, **kw)
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32 and tokens.shape == logprobs.shape == u.shape
    assert torch.equal(tokens, qlinear.sample(x, u, **kw))
    each = {k: v.double().tolist() if isinstance(v, torch.Tensor) else [v] * x.shape[0] for k, v in kw.items()}
    V = x.shape[1]
    for b in range(x.shape[0]):
        token, logprob = definition(x[b], float(u[b]), *(each[k][b] if k != "top_k" else int(each[k][b]) for k in PLAIN))
        got = float(logprobs[b])
        assert int(tokens[b]) == token, (b, int(tokens[b]), token)
        if math.isnan(logprob):
            assert math.isnan(got)
        else:
            # fp32's rounding, the sum's rounding to multiples of 2^-S, a few steps of float64
            scale = min(46, 63 - (V - 1).bit_length())
            assert abs(got - logprob) <= 2.0 ** -24 * abs(logprob) + V * 2.0 ** -(scale + 1) + 1e-13 * (1 + abs(logprob)), (b, got, logprob)
    return tokens


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.6, top_p=0.9), dict(temperature=1.7, top_p=0.99), dict(top_k=1),
            dict(top_k=7, temperature=0.8), dict(top_k=600, top_p=0.7), dict(min_p=0.1), dict(top_k=50, top_p=0.95, min_p=0.02),
            dict(top_p=0.0), dict(top_p=0.3, temperature=3.0), dict(temperature=100.0, top_p=0.999)]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("V", [1, 2, 7, 33, 512, 1000, 4097, 32003, 128256])
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_settings_and_sizes(dtype, V, settings):
    g = gen(V)
    x = (torch.randn(5, V, generator=g, device="cuda") * 2.5).to(dtype)
    check(x, torch.rand(5, generator=g, device="cuda"), **settings)


@pytest.mark.parametrize("dtype,V", [(BF, 262145), (F32, 200001), (HF, 655104), (F32, 327552)])
def test_long_rows(dtype, V):
    """More tokens than 2^17 (a coarser unit of the weights), up to the longest row."""
    g = gen(V)
    x = (torch.randn(3, V, generator=g, device="cuda") * 2).to(dtype)
    u = torch.rand(3, generator=g, device="cuda")
    for s in (dict(), dict(top_p=0.95), dict(top_k=100, min_p=0.01)):
        check(x, u, **s)
    with pytest.raises(qlinear.QlError):
        qlinear.sample(torch.zeros(1, 655105, dtype=HF, device="cuda"), u[:1])


@pytest.mark.parametrize("rows", [1, 2, 37, 148, 300, 1200])
@pytest.mark.parametrize("V", [40, 5000, 50257])
def test_batches_with_settings_of_their_own(rows, V):
    g = gen(rows + V)
    rand = lambda: torch.rand(rows, generator=g, device="cuda")  # noqa: E731
    x = (torch.randn(rows, V, generator=g, device="cuda") * 2).to(BF)
    own = dict(temperature=torch.where(rand() < 0.2, 0.0, 0.3 + rand()), top_k=torch.where(rand() < 0.4, 0, 1 + 1500 * rand()).int(),
               top_p=torch.where(rand() < 0.3, 1.0, rand()), min_p=torch.where(rand() < 0.5, 0.0, 0.2 * rand()))
    u = rand()
    tokens = check(x[:200], u[:200], **{k: v[:200].contiguous() for k, v in own.items()})
    # a row's token does not depend on the batch, its order, or how the batch divides a row
    whole = qlinear.sample(x, u, **own)
    assert torch.equal(whole[:200], tokens)
    back = torch.arange(rows - 1, -1, -1, device="cuda")
    assert torch.equal(qlinear.sample(x[back], u[back], **{k: v[back] for k, v in own.items()})[back], whole)
    one = rows // 2
    assert torch.equal(qlinear.sample(x[one:one + 1], u[one:one + 1], **{k: v[one:one + 1] for k, v in own.items()}), whole[one:one + 1])


@pytest.mark.parametrize("settings", [dict(top_p=0.9, temperature=1.3), dict(top_p=0.98), dict(top_k=3000, top_p=0.8), dict(top_k=400)], ids=str)
def test_many_rows_of_distinct_logits(settings):
    """Every logit its own value: some lie on the borders of whatever the rows are divided by on the way."""
    g = gen(60)
    x = torch.randn(300, 60001, generator=g, device="cuda") * 2
    check(x, torch.rand(300, generator=g, device="cuda"), **settings)


@pytest.mark.parametrize("far", [0.0, 1e4, -3e6])
@pytest.mark.parametrize("std", [1e-3, 1.0, 300.0])
def test_narrow_and_wide_rows_far_from_zero(far, std):
    """Logits whose spread is small next to their size, or large next to the temperature."""
    g = gen(70)
    x = far + torch.randn(20, 20011, generator=g, device="cuda") * std
    u = torch.rand(20, generator=g, device="cuda")
    for s in (dict(top_p=0.9), dict(top_k=1500, top_p=0.7), dict(top_k=40, top_p=0.9), dict(top_p=0.5, temperature=max(std, 1e-3)), dict()):
        check(x, u, **s)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [64, 1000, 16384, 100000])
def test_equal_logits(dtype, V):
    """All weights 1: borders are whole numbers, the prefix of n tokens is the first n indices."""
    x = torch.full((8, V), 3.25, dtype=dtype, device="cuda")
    u = torch.arange(8, device="cuda") / 8
    want = torch.arange(8, device="cuda") * V // 8
    assert torch.equal(check(x, u), want)
    for n in (1, 3, V // 4, V // 2):
        assert torch.equal(check(x, u, top_k=n), torch.arange(8, device="cuda") * n // 8)
    assert torch.equal(check(x, u, top_p=0.5), torch.arange(8, device="cuda") * (V // 2) // 8)
    assert torch.equal(check(x, u, top_k=V // 2, top_p=0.25), torch.arange(8, device="cuda") * (V // 8) // 8)
    check(x, u, min_p=1.0)
    check(x, u, temperature=0.0)


@pytest.mark.parametrize("top_k", [0, 300, 5000, 20000])
@pytest.mark.parametrize("top_p", [1.0, 0.6])
def test_few_different_values(top_k, top_p):
    """Thousands of equal logits at the border: the lowest indices stay."""
    g = gen(top_k)
    x = torch.randint(-3, 4, (6, 30000), generator=g, device="cuda").to(BF) / 2
    check(x, torch.rand(6, generator=g, device="cuda"), top_k=top_k, top_p=top_p)
    x = torch.where(torch.rand(6, 30000, generator=g, device="cuda") < 0.5, 0.0, -0.0)  # the same value
    check(x, torch.rand(6, generator=g, device="cuda"), top_k=top_k, top_p=top_p)
    check(x, torch.rand(6, generator=g, device="cuda"), temperature=0.0)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_masked_and_infinite_logits(dtype):
    g = gen(5)
    x = (torch.randn(9, 5000, generator=g, device="cuda") * 2).to(dtype)
    x[0] = -math.inf                       # nothing to draw
    x[1, 17] = math.nan
    x[2, 5:] = -math.inf                   # five left
    x[3] = -math.inf
    x[3, 4999] = -1e4                      # one left, a very low one
    x[4, [7, 4000]] = math.inf             # two share everything
    x[5, :2500] = torch.finfo(dtype).min   # the type's lowest value: as good as masked beside others
    x[6] = torch.finfo(dtype).min          # .. and the same for all without them
    x[7, 3] = torch.finfo(dtype).max
    x[8, 11] = -math.nan
    u = torch.rand(9, generator=g, device="cuda")
    for s in SETTINGS:
        t = check(x, u, **s)
        assert t[[0, 1, 8]].tolist() == [-1] * 3 and int(t[3]) == 4999 and int(t[4]) in (7, 4000) and int(t[7]) == 3
    # more kept than there are above -inf
    check(x, u, top_k=4000)


def test_extreme_settings():
    g = gen(6)
    x = torch.randn(6, 3000, generator=g, device="cuda")
    u = torch.rand(6, generator=g, device="cuda")
    greedy = x.argmax(-1)
    for t in (1e-30, 1e-320, 1e-5):
        assert torch.equal(qlinear.sample(x, u, temperature=t), greedy)
    for t in (1e30, math.inf):
        assert torch.equal(qlinear.sample(x, u, temperature=t), (u.double() * 3000).long())
    # u outside [0, 1) and not a number, settings that are not numbers, a negative temperature in a vector
    t = check(x, torch.tensor([0.0, 1.0, 5.0, -1.0, math.nan, math.inf], device="cuda"), top_k=10)
    assert int(t[4]) == -1
    nan = torch.tensor([1.0, math.nan, 1.0, 1.0, 1.0, 1.0], device="cuda")
    for k in ("temperature", "top_p", "min_p"):
        assert (check(x, u, **{**PLAIN, k: nan}) == -1).tolist() == [False, True] + [False] * 4
    assert (check(x, u, temperature=-nan) == -1).all()
    # vectors take what numbers refuse as their end: no filter, the largest alone
    every = torch.ones(6, device="cuda")
    assert torch.equal(qlinear.sample(x, u, top_k=(-3 * every).int(), top_p=2 * every, min_p=-every), qlinear.sample(x, u))
    assert torch.equal(qlinear.sample(x, u, min_p=3 * every), greedy) and torch.equal(qlinear.sample(x, u, top_p=-every), greedy)


def test_random_numbers_at_the_borders():
    """Four tokens of weights 1, 1/2, 1/4, 1/4 in another order: u exactly on a border takes the next."""
    ln2 = math.log(2)
    x = torch.tensor([[-2 * ln2, 0.0, -2 * ln2, -ln2]], dtype=torch.float64).float().cuda().expand(5, 4)
    # (fp32 logits: the weights are those within 2^-23, so the borders are approached from both sides)
    for d in (-1e-6, 1e-6):
        u = torch.tensor([0.125, 0.625, 0.75, 0.999, 0.0], device="cuda") + d
        check(x, u)
    exact = torch.zeros(5, 4, device="cuda")
    assert check(exact, torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")).tolist() == [0, 1, 2, 3, 3]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strides_and_alignment(dtype, shift):
    """Rows of a wider tensor, off the 16-byte grid, of an odd length, shared by all draws, transposed."""
    g = gen(shift)
    wide = (torch.randn(7, 5003, generator=g, device="cuda") * 2).to(dtype)
    u = torch.rand(7, generator=g, device="cuda")
    s = dict(top_k=100, top_p=0.9)
    x = wide[:, shift:shift + 4001]
    a = check(x, u, **s)
    assert torch.equal(a, check(x.contiguous(), u, **s))
    b = check(wide[2:3, shift:].expand(7, -1), u, **s)
    assert torch.equal(b, check(wide[2:3, shift:].repeat(7, 1), u, **s))
    assert torch.equal(a, check(x.t().contiguous().t(), u, **s))
    # what lies beside the rows is not read
    wide[:, :shift] = math.inf
    wide[:, shift + 4001:] = math.nan
    assert torch.equal(a, check(x, u, **s))


def test_many_rows_and_offsets_past_32_bits():
    g = gen(7)
    x = torch.randn(70001, 5, generator=g, device="cuda")
    u = torch.rand(70001, generator=g, device="cuda")
    got = qlinear.sample(x, u)
    w = (x.double() - x.double().max(-1, keepdim=True).values).exp().cumsum(-1)
    assert torch.equal(got, (w <= u.double()[:, None] * w[:, -1:]).sum(-1))
    big = torch.empty(36000, 128256, dtype=BF, device="cuda")  # 4.6e9 logits
    big[-3:] = (torch.randn(3, 128256, generator=g, device="cuda") * 2).to(BF)
    big[:-3] = 0
    got = qlinear.sample(big, u[:36000], top_p=0.9)
    assert torch.equal(got[-3:], check(big[-3:].clone(), u[35997:36000], top_p=0.9))
    # (all equal: the first nine tenths stay)
    kept = math.ceil(0.9 * 128256)
    assert torch.equal(got[:-3], (u[:35997].double() * kept).long())


def test_empty_batch():
    assert qlinear.sample(torch.zeros(0, 50, device="cuda"), torch.zeros(0, device="cuda")).shape == (0,)


def test_streams_graphs_and_two_calls_at_once():
    g = gen(8)
    x = (torch.randn(40, 128256, generator=g, device="cuda") * 2).to(BF)
    u = torch.rand(40, generator=g, device="cuda")
    call = lambda: qlinear.sample(x, u, temperature=0.9, top_k=2000, top_p=0.95)  # noqa: E731
    first = call()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs += [call() for _ in range(4)]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(first, o) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    out.zero_()
    graph.replay()
    assert torch.equal(first, out)
    u.copy_(torch.rand(40, generator=g, device="cuda"))  # a replay draws with the numbers of its time
    graph.replay()
    assert torch.equal(out, call())


def test_refusals(dev):
    x, u = torch.zeros(3, 10, device=dev), torch.zeros(3, device=dev)
    for bad in (dict(logits=x[0]), dict(logits=x[:, :0]), dict(logits=x.double()), dict(logits=x.cpu()), dict(u=u[:2]), dict(u=u.double()),
                dict(u=u.cpu()), dict(u=torch.zeros(6, device=dev)[::2]), dict(u=None), dict(temperature=-1.0), dict(temperature=math.nan),
                dict(top_k=-1), dict(top_k=1.5), dict(top_p=-0.1), dict(min_p=1.5), dict(min_p=-0.5), dict(top_k=u), dict(top_p=u[:2]),
                dict(temperature=u.half()), dict(min_p=u.cpu()), dict(temperature="hot")):
        a = {**dict(logits=x, u=u), **bad}
        with pytest.raises((ValueError, TypeError)):
            qlinear.sample(a.pop("logits"), a.pop("u"), **a)
