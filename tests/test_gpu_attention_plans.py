"""GPU: paged attention under every division of the work -- one piece, splits joined in a cluster,
pieces sized by the lengths, pieces of 2048 joined by a second launch, the tensor-core kernel whole
and split, and batches that mix the two kernels."""
import math

import pytest
import torch

import qlinear
from qlinear import _lib
from test_gpu_decoder import BF, HF, U, attention_reference, check_attention, gen, paged, rnd, within

pytestmark = pytest.mark.gpu

# new tokens, lengths, q heads, kv heads, head size, whether partial results go through memory
PLANS = {
    "one piece": ([1, 1], [100, 20], 4, 2, 128, False),
    "cluster": ([1, 2], [900, 300], 6, 2, 64, False),
    "cluster, 256": ([40], [300], 4, 2, 256, False),
    "by lengths": ([1, 1], [9000, 7000], 4, 2, 128, True),
    "by lengths, 96": ([80], [7000], 4, 2, 96, True),
    "pieces": ([1] * 40, [5000, 1, 3000, 20] * 10, 4, 2, 64, True),
    "tiles": ([200], [300], 6, 2, 128, False),
    "tiles, 64": ([200], [300], 6, 2, 64, False),
    "tiles, split": ([200], [9000], 6, 2, 128, True),
    "tiles, 64, split": ([200], [9000], 6, 2, 64, True),
    "mixed": ([1, 200, 1], [9000, 300, 20], 6, 2, 128, True),
}


def planned(plan):
    q_lens, kv_lens, Hq, Hkv, D, split = PLANS[plan]
    need = qlinear.paged_attention_workspace_size(sum(q_lens), Hq, Hkv, D, len(q_lens), max(q_lens), max(kv_lens))
    assert (need > 0) == split, plan
    return q_lens, kv_lens, Hq, Hkv, D


# ------------------------------------------------------------------------ values that are not finite

@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_query_that_is_not_finite(plan, dtype, value):
    """A query with a NaN (or an infinity, whose scores have a maximum of infinity) gives NaN and
    not the zeros of a token that sees nothing; every other row is as before."""
    q_lens, kv_lens, Hq, Hkv, D = planned(plan)
    g = gen(len(plan))
    q, kc, vc, table, starts, lens = paged(g, q_lens, kv_lens, Hq, Hkv, D, 16, dtype)
    o, a = attention_reference(q, kc, vc, table, q_lens, kv_lens, D ** -0.5, True, 0)
    hit = [(0, Hq - 1)] + ([(sum(q_lens) - 1, 0)] if sum(q_lens) > 1 else [])  # each sees 20 positions at least
    q = q.clone()
    for t, h in hit:
        q[t, h, D // 3] = value
    got = qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=max(q_lens), max_kv=max(kv_lens))
    ok = torch.ones(got.shape[:2], dtype=torch.bool, device="cuda")
    for t, h in hit:
        assert got[t, h].isnan().all(), (t, h)
        ok[t, h] = False
    # weights and output rounded once to the dtype; scores below 2^7, so their fp32 rounding moves
    # an exponent by 2^-24 * 64 * 2^7 at most; f16 weights under 2^-14 lose 2^-25 each
    e = 2.0 ** -24 * 64 * 2 ** 7
    low = max(kv_lens) * 2.0 ** -25 * 8 if dtype == HF else 0.0
    within(got[ok], o[ok], (U[dtype] * (a + o.abs()) + 2 * e * a + low)[ok])
    assert qlinear.device_error() == 0


@pytest.mark.parametrize("plan", PLANS)
def test_key_that_is_not_a_number(plan):
    """A NaN key reaches exactly the rows that see its position: all heads of its group, from its
    token on."""
    q_lens, kv_lens, Hq, Hkv, D = planned(plan)
    g = gen(len(plan))
    q, kc, vc, table, starts, lens = paged(g, q_lens, kv_lens, Hq, Hkv, D, 16, BF)
    o, a = attention_reference(q, kc, vc, table, q_lens, kv_lens, D ** -0.5, True, 0)
    at = max(0, kv_lens[0] - (q_lens[0] + 1) // 2)  # within the first sequence's new tokens
    kc[table[0, at // 16].long(), Hkv - 1, at % 16, 5] = math.nan
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    first = at - (kv_lens[0] - q_lens[0])
    bad[first:q_lens[0], Hq - Hq // Hkv:] = True
    got = qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=max(q_lens), max_kv=max(kv_lens))
    assert bad.any() and got[bad].isnan().all()
    within(got[~bad], o[~bad], (U[BF] * (a + o.abs()) + 2 * 2.0 ** -24 * 64 * 2 ** 7 * a)[~bad])


# ------------------------------------------------------------------------ f16 weights

@pytest.mark.parametrize("D,Hkv,T", [(64, 8, 16384), (128, 8, 16384), (256, 8, 16384), (128, 1, 1)])
def test_f16_keeps_the_weight_of_a_long_tail(D, Hkv, T):
    """One score above 524287 others by so much that each of them weighs 2^-24.9 of it: together 1.7 %
    of the sum, each half a step of f16's smallest numbers.  With every value 1 the result is 1."""
    n, ps = 524288, 128
    kc = torch.zeros(n // ps, Hkv, ps, D, dtype=HF, device="cuda")
    vc = torch.ones_like(kc)
    kc[0, :, 0, 0] = 24.91 * math.log(2)
    q = torch.zeros(T, Hkv, D, dtype=HF, device="cuda")
    q[..., 0] = 1
    i32 = dict(dtype=torch.int32, device="cuda")
    got = qlinear.paged_attention(q, kc, vc, torch.arange(n // ps, **i32)[None], torch.tensor([0, T], **i32), torch.tensor([n], **i32),
                                  max_q=T, max_kv=n, scale=1.0, causal=False)
    # the output's rounding (2^-11), and at most 2^-23 of the fp32 accumulator in each product of 16
    # positions, of which a piece with the high score has up to 131072 for a warp or tile
    assert float((got.double() - 1).abs().max()) <= 2.0 ** -11 + 131072 / 16 * 2.0 ** -23
    assert qlinear.device_error() == 0


# ------------------------------------------------------------------------ long chunks

@pytest.mark.parametrize("D", [64, 96, 128])
def test_chunk_of_more_than_a_million_rows(D):
    """70000 tokens of 16 heads on one kv head, each seeing 50 positions."""
    n, H, W, ps = 70000, 16, 50, 64
    g = gen(D)
    q, cache = rnd(g, n, H, D), rnd(g, -(-n // ps), 2, ps, D)
    kc, vc = cache[:, :1], cache[:, 1:]
    i32 = dict(dtype=torch.int32, device="cuda")
    got = qlinear.paged_attention(q, kc, vc, torch.arange(-(-n // ps), **i32)[None], torch.tensor([0, n], **i32), torch.tensor([n], **i32),
                                  max_q=n, max_kv=n, window=W)
    at = torch.cat([torch.arange(64), torch.arange(64, n, 61), torch.arange(n - 64, n)]).cuda()
    pos = at[:, None] - W + 1 + torch.arange(W, device="cuda")
    k, v = (c.reshape(-1, D)[pos.clamp(min=0)].double() for c in (kc, vc))
    s = torch.einsum("ihd,ijd->ihj", q[at].double(), k) * D ** -0.5
    p = s.masked_fill((pos < 0)[:, None], -math.inf).softmax(-1)
    o, a = torch.einsum("ihj,ijd->ihd", p, v), torch.einsum("ihj,ijd->ihd", p, v.abs())
    within(got[at], o, U[BF] * (a + o.abs()) + 2 * 2.0 ** -24 * 64 * 2 ** 7 * a)
    assert qlinear.device_error() == 0


# ------------------------------------------------------------------------ waits that run out under way

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_len,kv", [(4096, 4096), (200, 9000), (400, 700), (130, 130)])
def test_loader_that_stops_half_way(D, q_len, kv):
    """With half of each CTA's loads (a flag that only this sets) and the wait limit at 20 ms, a launch
    that has products and copies behind it ends by itself and says so, and the next call is right."""
    g = gen(D + kv)
    q, kc, vc, table, starts, lens = paged(g, [q_len], [kv], 6, 2, D, 16, BF)
    call = lambda: qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=q_len, max_kv=kv)  # noqa: E731
    want = call()
    assert qlinear.device_error() == 0
    try:
        _lib.debug_inject(_lib.INJECT_ATTENTION_PRODUCER_STOPS, 20_000_000)
        call()
        err = qlinear.device_error()
    finally:
        _lib.debug_inject(0, 0)
    assert err & (_lib.DEV_ERR_TIMEOUT_FULL | _lib.DEV_ERR_TIMEOUT_EMPTY | _lib.DEV_ERR_TIMEOUT_ACC)
    assert torch.equal(call(), want) and qlinear.device_error() == 0


# ------------------------------------------------------------------------ bounds that are too low

@pytest.mark.parametrize("D", [64, 256])
def test_a_bound_of_no_new_tokens_is_reported(D):
    """max_q = 0 with tokens there: the error word is set, as for every bound that is too low."""
    q, kc, vc, table, starts, lens = paged(gen(D), [1, 40], [10, 300], 6, 2, D, 16, BF)
    assert qlinear.device_error() == 0
    qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=0, max_kv=300)
    assert qlinear.device_error() == _lib.DEV_ERR_BAD_INDEX
    qlinear.paged_attention(q, kc, vc, table, torch.zeros_like(starts), lens, max_q=0, max_kv=300)  # no sequence has any
    assert qlinear.device_error() == 0


# ------------------------------------------------------------------------ every plan against 64 bits

@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_pieces_of_many_sequences(D, dtype):
    """More than 32 sequences over 2048 positions: fixed pieces, many of them empty."""
    kv = [1, 5000, 2048, 2049, 17, 4096, 4097, 300] * 5
    assert qlinear.paged_attention_workspace_size(40, 4, 2, D, 40, 1, 5000) > 0
    check_attention(gen(D), [1] * 40, kv, 4, 2, D, 64, dtype)


@pytest.mark.parametrize("D,causal,window", [(64, True, 0), (128, True, 0), (128, False, 0), (128, True, 3000), (256, True, 0)])
def test_pieces_under_a_bound_far_above_the_lengths(D, causal, window):
    """A bound of 140000 positions (what a captured graph is given): 64 longer pieces, nearly all empty."""
    q_lens, kv, bound = [1] * 40, [1, 4000, 2600, 700] * 10, 140000
    g = gen(D + window)
    q, kc, vc, table, starts, lens = paged(g, q_lens, kv, 4, 2, D, 64, BF)
    wide = torch.full((40, -(-bound // 64)), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    got = qlinear.paged_attention(q, kc, vc, wide, starts, lens, max_q=1, max_kv=bound, causal=causal, window=window)
    o, a = attention_reference(q, kc, vc, table, q_lens, kv, D ** -0.5, causal, window)
    within(got, o, U[BF] * (a + o.abs()) + 2 * 2.0 ** -24 * 64 * 2 ** 7 * a)
    assert qlinear.device_error() == 0


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kv,window", [([20011], 0), ([7000, 1], 0), ([9000, 12001, 6400], 0), ([20011, 300, 7001], 6500)])
def test_pieces_by_lengths(D, dtype, kv, window):
    """A few sequences over 6000 positions: the kernel divides them by their lengths."""
    assert qlinear.paged_attention_workspace_size(len(kv), 6, 2, D, len(kv), 1, max(kv), window) > 0
    check_attention(gen(D + len(kv)), [1] * len(kv), kv, 6, 2, D, 32, dtype, True, window)


@pytest.mark.parametrize("kv", [[700, 130, 2, 1], [5000], [9000, 6100], [12000] * 3])
@pytest.mark.parametrize("D,causal,window", [(64, False, 0), (128, False, 0), (64, True, 1), (128, True, 100), (128, True, 2500)])
def test_single_tokens_with_masks(kv, D, causal, window):
    check_attention(gen(window + len(kv)), [1] * len(kv), kv, 4, 2, D, 16, BF, causal, window)


@pytest.mark.parametrize("D", [64, 96, 256])
@pytest.mark.parametrize("q_len", [2, 150])
def test_long_contexts_of_other_head_sizes(D, q_len):
    check_attention(gen(D + q_len), [q_len, q_len], [9001, 1000], 6, 2, D, 64)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_clusters_of_eight(D, dtype):
    """One sequence of up to 6000 positions: eight splits, with heads of 256 each CTA alone on its SM."""
    assert qlinear.paged_attention_workspace_size(1, 6, 2, D, 1, 1, 6000) == 0
    for kv, window in (([6000], 0), ([5999], 1500), ([1100], 0)):
        check_attention(gen(D + kv[0]), [1], kv, 6, 2, D, 16, dtype, True, window)
