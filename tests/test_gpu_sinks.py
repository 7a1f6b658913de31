"""GPU: attention over a window with sinks, against 64 bits, under every division of the work; the poisoned places
and table entries of test_gpu_decoder's caches, and the pages between the sinks and the windows given back."""
import math

import pytest
import torch

import qlinear
from qlinear import _lib
from test_gpu_decoder import BF, HF, U, gen, paged, rnd, within

pytestmark = pytest.mark.gpu


def evicted(kc, vc, table, q_lens, kv_lens, window, sinks):
    """The pages that no new token sees poisoned, their table entries past the cache."""
    ps = kc.shape[2]
    table = table.clone()
    for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
        first = max(0, L - n + 1 - window)
        for i in range(-(-sinks // ps), first // ps):
            page = int(table[b, i])
            kc[page], vc[page] = math.nan, math.inf
            table[b, i] = 1 << 30
    return table


def reference(q, kc, vc, table, q_lens, kv_lens, window, sinks):
    """(o, softmax @ |v|) in 64 bits over the positions that some token sees."""
    T, Hq, D = q.shape
    Hkv, ps = kc.shape[1], kc.shape[2]
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    at = 0
    for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
        if n and L:
            first = max(0, L - n + 1 - window)
            j = torch.cat([torch.arange(min(sinks, first, L)), torch.arange(min(first, L), L)]).to(q.device)
            pages = table[b].long()[j // ps]
            k, v = (c[pages, :, j % ps].double().repeat_interleave(Hq // Hkv, 1) for c in (kc, vc))
            s = torch.einsum("ihd,jhd->hij", q[at:at + n].double(), k) * D ** -0.5
            i = torch.arange(n, device=q.device)[:, None] + (L - n)
            see = (j <= i) & ((j > i - window) | (j < sinks))
            p = torch.softmax(s.masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
            o[at:at + n] = torch.einsum("hij,jhd->ihd", p, v)
            a[at:at + n] = torch.einsum("hij,jhd->ihd", p, v.abs())
        at += n
    return o, a


def check(g, q_lens, kv_lens, Hq, Hkv, D, window, sinks, ps=16, dtype=BF, max_kv=None):
    q, kc, vc, table, starts, lens = paged(g, q_lens, kv_lens, Hq, Hkv, D, ps, dtype)
    o, a = reference(q, kc, vc, table, q_lens, kv_lens, window, sinks)
    given_back = evicted(kc, vc, table, q_lens, kv_lens, window, sinks)
    max_kv = max_kv or max(kv_lens)
    given_back = torch.nn.functional.pad(given_back, (0, -(-max_kv // ps)), value=-1)
    got = qlinear.paged_attention(q, kc, vc, given_back, starts, lens, max_q=max(q_lens), max_kv=max_kv, window=window, sinks=sinks)
    # weights rounded to the dtype and the output (U each); scores below 2^7: their fp32 rounding moves an
    # exponent by 2^-24 * 64 * 2^7 at most; f16 weights under 2^-14 lose 2^-25 each
    e = 2.0 ** -24 * 64 * 2 ** 7
    low = max(kv_lens) * 2.0 ** -25 * 8 if dtype == HF else 0.0
    within(got, o, U[dtype] * (a + o.abs()) + 2 * e * a + low, "o")
    assert qlinear.device_error() == 0
    return got


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 4), (37, 16), (100, 70), (128, 128), (300, 1), (300, 200), (64, 1024), (100000, 4)])
def test_single_tokens(D, dtype, window, sinks):
    """Lengths inside the window, just past it, and where sinks and window touch."""
    kv = [1, 2, 17, sinks, sinks + 1, window % 1000 + 1, sinks + window % 1000, sinks + window % 1000 + 1, sinks + window % 1000 + 40, 2000]
    check(gen(D + sinks), [1] * len(kv), kv, 6, 2, D, window, sinks, dtype=dtype)


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 24, 8), (64, 8, 8), (128, 7, 1), (64, 3, 1), (96, 6, 2), (256, 4, 2)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("window,sinks", [(1, 1), (40, 4), (128, 128), (129, 130), (70, 300), (200, 37), (1000, 4)])
def test_chunks(D, Hq, Hkv, dtype, window, sinks):
    """Sinks and windows that begin and end inside tiles of 16 and 128, apart and touching; sequences
    without new tokens, shorter than the sinks, and a first chunk."""
    q = [1, 17, 128, 0, 200, 85, 3, 257, 300]
    kv = [512, 17, 129, 50, 200, 1000, 400, 900, 2111]
    check(gen(D + window), q, kv, Hq, Hkv, D, window, sinks, 32, dtype)


@pytest.mark.parametrize("ps", [16, 64, 128, 512, 1024])
@pytest.mark.parametrize("q_len", [1, 150])
def test_page_sizes(ps, q_len):
    for window, sinks in ((100, 4), (600, 130)):
        check(gen(ps), [q_len, q_len], [3000, 1500], 6, 2, 128, window, sinks, ps)


@pytest.mark.parametrize("q_lens,kv_lens,Hq,Hkv,D,window", [
    ([1], [3000], 6, 2, 128, 900),               # splits joined in a cluster
    ([1, 1], [40000, 20000], 4, 2, 128, 9000),   # pieces by the lengths
    ([1] * 40, [9000, 1, 3000, 20] * 10, 4, 2, 64, 5000),  # pieces of 2048
    ([40], [9000], 4, 2, 256, 7000), ([80], [9000], 4, 2, 96, 7000),
    ([200], [20000], 6, 2, 128, 9000), ([200], [20000], 6, 2, 64, 9000),  # tiles, split
    ([1, 200, 1], [20000, 300, 20], 6, 2, 128, 9000),  # both kernels
])
@pytest.mark.parametrize("sinks", [1, 4, 64, 200, 1024])
def test_divisions(q_lens, kv_lens, Hq, Hkv, D, window, sinks):
    for shift in (0, 5, 64, 127):  # where in a tile the window begins
        check(gen(sinks + shift), q_lens, [max(n, k - shift) for n, k in zip(q_lens, kv_lens)], Hq, Hkv, D, window, sinks, max_kv=max(kv_lens))


def test_rows_that_see_nothing():
    """kv_len 0, and more new tokens than cached positions."""
    for D in (64, 128):
        got = check(gen(D), [3, 5, 40, 4], [0, 2, 9, 4], 6, 2, D, 3, 2)
        assert not got[:3].any() and not got[3:6].any() and got[6:8].any()
        check(gen(D), [3, 300], [0, 200], 6, 2, D, 20, 7)


def test_wide_windows_are_plain_attention():
    """A window that holds everything, and sinks up to the window: the same as without."""
    q, kc, vc, table, starts, lens = paged(gen(3), [1, 60], [90, 300], 6, 2, 128, 16, BF)
    call = lambda **kw: qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=60, max_kv=300, **kw)  # noqa: E731
    assert torch.equal(call(), call(window=300, sinks=5))
    assert torch.equal(call(), call(window=10 ** 6, sinks=1024))
    o, a = reference(q, kc, vc, table, [1, 60], [90, 300], 200, 100)
    within(call(window=200, sinks=100), o, U[BF] * (a + o.abs()) + 2 * 2.0 ** -24 * 64 * 2 ** 7 * a)


@pytest.mark.parametrize("q_len", [1, 150])
def test_values_that_are_not_finite(q_len):
    """A NaN key among the sinks reaches every row of its head, one between sinks and windows none."""
    q, kc, vc, table, starts, lens = paged(gen(4), [q_len], [3000], 4, 2, 128, 16, BF)
    o, a = reference(q, kc, vc, table, [q_len], [3000], 500, 20)
    kc[table[0, 60].long()] = math.nan   # positions 960 - 975
    vc[table[0, 60].long()] = math.nan
    kc[table[0, 1].long(), 1, 3, 9] = math.nan  # position 19 of the second head
    got = qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=q_len, max_kv=3000, window=500, sinks=20)
    assert got[:, 2:].isnan().all()
    within(got[:, :2], o[:, :2], (U[BF] * (a + o.abs()) + 2 * 2.0 ** -24 * 64 * 2 ** 7 * a)[:, :2])


@pytest.mark.parametrize("q_lens", [[1] * 5, [1, 70, 1, 200, 3]])
def test_streams_and_graphs(q_lens):
    g = gen(5)
    kv = [a + b for a, b in zip(q_lens, [3000, 5, 2000, 0, 77])]
    q, kc, vc, table, starts, lens = paged(g, q_lens, kv, 6, 2, 128, 16, BF)
    table = torch.nn.functional.pad(table, (0, 8192 // 16 - table.shape[1]), value=-1)
    call = lambda: qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=max(q_lens), max_kv=8192, window=700, sinks=33)  # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    out.zero_()
    graph.replay()
    assert torch.equal(first, out)
    lens -= torch.tensor([1100, 0, 700, 0, 1], dtype=torch.int32, device="cuda")
    graph.replay()
    shorter = lens.tolist()
    o, a = reference(q, kc, vc, table, q_lens, shorter, 700, 33)
    within(out, o, U[BF] * (a + o.abs()) + 2 * 2.0 ** -24 * 64 * 2 ** 7 * a)
    assert qlinear.device_error() == 0


def test_offsets_past_32_bits():
    """Sinks and window in pages whose element offset exceeds 2^31."""
    P, Hkv, ps, D = 135_000, 8, 16, 128
    cache = torch.empty(P, Hkv, ps, D, dtype=BF, device="cuda")
    pages = [P - 1, 3, P - 70, 131_072]
    cache[torch.tensor(pages, device="cuda")] = rnd(gen(2), 4, Hkv, ps, D)
    table = torch.full((1, 400), -1, dtype=torch.int32)
    table[0, 0], table[0, 397:400] = pages[0], torch.tensor(pages[1:], dtype=torch.int32)
    table = table.cuda()
    for n, window in ((1, 40), (20, 20)):
        q = rnd(gen(n), n, 16, D)
        starts, lens = torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.tensor([6399], dtype=torch.int32, device="cuda")
        got = qlinear.paged_attention(q, cache, cache, table, starts, lens, max_q=n, max_kv=6399, window=window, sinks=9)
        o, a = reference(q, cache, cache, table, [n], [6399], window, 9)
        within(got, o, U[BF] * (a + o.abs()) + 2 * 2.0 ** -24 * 64 * 2 ** 7 * a)
    assert qlinear.device_error() == 0


def test_refusals(dev):
    q, kc, vc, table, starts, lens = paged(gen(7), [1, 2], [10, 20], 4, 2, 64, 16, BF)
    call = lambda **kw: qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=2, max_kv=20, **kw)  # noqa: E731
    for bad in (dict(sinks=4), dict(window=4, sinks=-1), dict(window=4, sinks=1025), dict(window=30, sinks=1025), dict(window=-4, sinks=4)):
        with pytest.raises(qlinear.QlError):
            call(**bad)
    with pytest.raises(ValueError):
        call(window=4, sinks=4, causal=False)
    with pytest.raises(TypeError):
        call(window=4, sinks=None)


def test_wait_runs_out_and_reports():
    """The loader with sinks stopped half-way: the launch ends by itself and the next call is right."""
    q, kc, vc, table, starts, lens = paged(gen(9), [200], [3000], 6, 2, 128, 16, BF)
    assert qlinear.device_error() == 0
    try:
        _lib.debug_inject(_lib.INJECT_ATTENTION_PRODUCER_STOPS, 50_000_000)
        qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=200, max_kv=3000, window=700, sinks=40)
        err = qlinear.device_error()
    finally:
        _lib.debug_inject(0, 0)
    assert err & (_lib.DEV_ERR_TIMEOUT_FULL | _lib.DEV_ERR_TIMEOUT_EMPTY | _lib.DEV_ERR_TIMEOUT_ACC)
    check(gen(10), [200], [3000], 6, 2, 128, 700, 40)
