"""GPU: the decoder operators (residual norm, rotary positions and the append, paged attention,
page copies) against plain 64-bit forms.

Tolerances follow from the arithmetic: every output is rounded once (unit roundoff u of its
dtype), everything before is fp32, and attention rounds its weights to the dtype (another u on
each weight) before the product with v."""
import math

import pytest
import torch

import qlinear
from qlinear import _lib

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}  # rounding of subnormals
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rnd(g, *shape, dtype=BF, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, bound, what=""):
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst excess "
                           f"{float(((got.double() - want).abs() - bound).nan_to_num(math.inf).max()):.3e}")


# ------------------------------------------------------------------------ residual norm

def norm_reference(y, res, w, post, gate, gp, alpha, scale, sp, eps, off):
    y, r = y.double(), res.double()
    M, D = y.shape
    row = lambda t, p: t.double().reshape(-1, D)[torch.arange(M, device=y.device) // p if p else torch.zeros(M, dtype=torch.long, device=y.device)]  # noqa: E731
    u = y
    if post is not None:
        u = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * (off + post.double())
    if gate is not None:
        u = u * row(gate, gp)
    size = r.abs() + abs(alpha) * u.abs()  # fp32 rounding of the sum is relative to its terms
    r = r + alpha * u
    f = (off + w.double()) / (r.square().mean(-1, keepdim=True) + eps).sqrt()
    if scale is not None:
        f = f * (1 + row(scale, sp))
    return r * f, r, size, f.abs()


def check_norm(y, res, w, post=None, gate=None, gp=0, alpha=1.0, scale=None, sp=0, eps=1e-5, off=0.0):
    h, r = qlinear.norm_residual(y, res, w, post_weight=post, gate=gate, gate_period=gp, alpha=alpha, scale=scale,
                                 scale_period=sp, eps=eps, weight_offset=off)
    D = y.shape[-1]
    wh, wr, size, f = norm_reference(y.reshape(-1, D), res.reshape(-1, D), w, post, gate, gp, alpha, scale, sp, eps, off)
    assert h.shape == y.shape and r.shape == y.shape and h.dtype == y.dtype and r.dtype == res.dtype
    # fp32: about 8 roundings on a value, a sum of D squares (error D * 2^-24 / 2 at worst, half of
    # it in the root), the reciprocal root's 2 ulp
    k = 2.0 ** -24 * (16 + D / 64)
    within(r.reshape(-1, D), wr, U[r.dtype] * wr.abs() + k * size + TINY[r.dtype], "r")
    within(h.reshape(-1, D), wh, U[h.dtype] * wh.abs() + 2 * k * (wh.abs() + f * size) + TINY[h.dtype], "h")


@pytest.mark.parametrize("dtype,rdtype", [(BF, BF), (HF, HF), (F32, F32), (BF, F32), (HF, F32)])
@pytest.mark.parametrize("M,D", [(1, 1), (1, 8), (3, 33), (5, 3072), (2, 4104), (300, 520), (2, 8191), (2, 20000), (1, 32768),
                                 (1, 32767)])
def test_norm_residual(dtype, rdtype, M, D):
    g = gen(M * 1000 + D)
    y, res = rnd(g, M, D, dtype=dtype), rnd(g, M, D, dtype=rdtype, std=3.0)
    w = (1 + rnd(g, D, dtype=F32, std=0.3)).to(dtype)
    check_norm(y, res, w)
    check_norm(y, res, w, post=(1 + rnd(g, D, dtype=F32, std=0.3)).to(dtype), gate=rnd(g, D, dtype=dtype), alpha=0.3,
               scale=rnd(g, D, dtype=dtype, std=0.3), off=0.0)


@pytest.mark.parametrize("D", [64, 61])
@pytest.mark.parametrize("gp,sp", [(0, 0), (7, 0), (3, 5), (1, 1)])
def test_norm_residual_periods_and_offset(D, gp, sp):
    g, M = gen(D + gp), 20
    rows = lambda p: -(-M // p) if p else 1  # noqa: E731
    check_norm(rnd(g, M, D), rnd(g, M, D), rnd(g, D, std=0.2), post=rnd(g, D, std=0.2), gate=rnd(g, rows(gp), D), gp=gp,
               alpha=-1.5, scale=rnd(g, rows(sp), D), sp=sp, off=1.0)


def test_norm_residual_strides_batches_and_zeros():
    g = gen(5)
    wide = rnd(g, 9, 3 * 64)
    check_norm(wide[:, 64:128], rnd(g, 9, 80)[:, :64], rnd(g, 64))          # rows inside a wider matrix
    check_norm(wide[:, 3:64], rnd(g, 9, 61), rnd(g, 61))                     # rows off the 16-byte grid
    check_norm(wide.t()[:64], rnd(g, 64, 9), rnd(g, 9))                      # a transposed view
    check_norm(rnd(g, 2, 3, 4, 64), rnd(g, 2, 3, 4, 64), rnd(g, 64))        # leading axes
    check_norm(rnd(g, 4, 64)[::2], rnd(g, 2, 64), rnd(g, 64))
    z = torch.zeros(3, 64, device="cuda", dtype=BF)
    h, r = qlinear.norm_residual(z, z, torch.ones(64, device="cuda", dtype=BF), post_weight=torch.ones(64, device="cuda", dtype=BF))
    assert not h.any() and not r.any()                                       # eps keeps the root finite
    h, r = qlinear.norm_residual(z[:0], z[:0], z[0])
    assert h.shape == (0, 64)
    y = rnd(g, 2, 64)
    y[0, 5] = math.inf  # a bad row stays in its row
    h, r = qlinear.norm_residual(y, z[:2], torch.ones(64, device="cuda", dtype=BF))
    assert not h[0].isfinite().all() and h[1].isfinite().all()


def test_norm_residual_refusals(dev):
    y = torch.zeros(4, 64, device=dev, dtype=BF)
    w = torch.zeros(64, device=dev, dtype=BF)
    for bad in (dict(residual=y[:3]), dict(weight=w[:32]), dict(weight=w.float()), dict(gate=torch.zeros(1, 64, device=dev, dtype=BF), gate_period=2),
                dict(scale=torch.zeros(128, 1, device=dev, dtype=BF)), dict(post_weight=w.cpu())):
        a = dict(residual=y, weight=w)
        a.update(bad)
        with pytest.raises((ValueError, TypeError)):
            qlinear.norm_residual(y, a.pop("residual"), a.pop("weight"), **a)
    with pytest.raises(qlinear.QlError):
        qlinear.norm_residual(y, y.half(), w)
    with pytest.raises(qlinear.QlError):
        big = torch.zeros(1, 32769, device=dev, dtype=BF)
        qlinear.norm_residual(big, big, big[0])
    with pytest.raises(qlinear.QlError):
        qlinear.norm_residual(y, y, w, gate=w, gate_period=-1)
    with pytest.raises(TypeError):
        qlinear.norm_residual(y.double(), y.double(), w.double())


# ------------------------------------------------------------------------ rotary positions

def rope_reference(x, table, positions, layout):
    x = x.double()
    rot = table.shape[1]
    row = table[positions].double()[:, None]
    cos, sin = row[..., :rot // 2], row[..., rot // 2:]
    out, size = x.clone(), x.abs().clone()
    i = torch.arange(rot // 2, device=x.device)
    ia, ib = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * cos - b * sin, b * cos + a * sin
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * table.abs().max().double()
    return out, size


def rope_bound(ref, size, dtype):
    return U[dtype] * ref.abs() + 2.0 ** -22 * size + TINY[dtype]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("T,Hq,Hk,D,rot", [(1, 24, 8, 128, 128), (7, 5, 1, 64, 32), (3, 3, 3, 96, 96), (2, 1, 0, 6, 2),
                                           (5, 2, 2, 80, 38), (4, 30, 30, 128, 128), (2, 2, 1, 256, 64), (9, 1, 1, 1024, 1024)])
def test_rope(layout, dtype, T, Hq, Hk, D, rot):
    g = gen(T + D)
    q, k = rnd(g, T, Hq, D, dtype=dtype), rnd(g, T, Hk, D, dtype=dtype)
    table = qlinear.rope_table(rot, 5000)
    pos = torch.randint(0, 5000, (T,), generator=g, device="cuda")
    pos[0] = 4999
    qo, ko = qlinear.rope(q, k, table, pos, layout=layout)
    for got, x in ((qo, q), (ko, k)):
        if x.numel():
            ref, size = rope_reference(x, table, pos, layout)
            within(got, ref, rope_bound(ref, size, dtype))
            assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_rope_append_strided_views(layout, off):
    """q, k, v as views of a fused projection (also off the 16-byte grid), a cache that is a
    plane of a larger pool, padding tokens, slots in any order; nothing else is written."""
    g = gen(11 + off)
    T, Hq, Hkv, D, ps, P = 21, 6, 2, 64, 16, 5
    qkv = rnd(g, T, (Hq + 2 * Hkv) * D + 16)[:, off:off + (Hq + 2 * Hkv) * D]
    q = qkv[:, :Hq * D].unflatten(1, (Hq, D))
    k = qkv[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D))
    v = qkv[:, (Hq + Hkv) * D:].unflatten(1, (Hkv, D))
    pool = rnd(g, 3, 2, P, Hkv, ps, D)
    before = pool.clone()
    table = qlinear.rope_table(D, 100)
    pos = torch.randint(0, 100, (T,), generator=g, device="cuda")
    slots = torch.randperm(P * ps, generator=g, device="cuda")[:T].clone()
    slots[4] = -1
    slots[20] = -7
    qo = qlinear.rope_append(q, k, v, table, pos, pool[1, 0], pool[1, 1], slots, layout=layout)
    ref, size = rope_reference(q, table, pos, layout)
    within(qo, ref, rope_bound(ref, size, BF))
    kref, ksize = rope_reference(k, table, pos, layout)
    want = before[1].transpose(2, 3).reshape(2, P * ps, Hkv, D).double()
    bound = torch.zeros_like(want)
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            want[0, s], want[1, s] = kref[t], v[t].double()
            bound[0, s] = rope_bound(kref, ksize, BF)[t]
    within(pool[1].transpose(2, 3).reshape(2, P * ps, Hkv, D), want, bound, "cache")
    assert torch.equal(pool[0], before[0]) and torch.equal(pool[2], before[2])
    assert qlinear.device_error() == 0


def test_rope_in_heads_first_layout():
    """A [heads, tokens, D] tensor viewed as [tokens, heads, D]."""
    g = gen(3)
    q = rnd(g, 4, 9, 64).transpose(0, 1)
    table = qlinear.rope_table(64, 9)
    pos = torch.arange(9, device="cuda")
    qo, ko = qlinear.rope(q, q[:, :1], table, pos)
    ref, size = rope_reference(q, table, pos, "half")
    within(qo, ref, rope_bound(ref, size, BF))
    within(ko, ref[:, :1], rope_bound(ref, size, BF)[:, :1])


def test_rope_bad_positions_and_slots_are_reported():
    g = gen(8)
    q, k = rnd(g, 3, 2, 64), rnd(g, 3, 1, 64)
    table = qlinear.rope_table(64, 10)
    assert qlinear.device_error() == 0
    qo, ko = qlinear.rope(q, k, table, torch.tensor([0, 10, -1], device="cuda"))
    assert qlinear.device_error() == _lib.DEV_ERR_BAD_INDEX
    assert torch.equal(qo[0], q[0]) and not qo[1:].any() and not ko[1:].any()
    kc, vc = rnd(g, 2, 1, 16, 64), rnd(g, 2, 1, 16, 64)
    k0, v0 = kc.clone(), vc.clone()
    qlinear.rope_append(q, k, k, table, torch.tensor([0, 10, 1], device="cuda"), kc, vc, torch.tensor([32, 3, -1], device="cuda"))
    assert qlinear.device_error() == _lib.DEV_ERR_BAD_INDEX
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


def test_rope_refusals(dev):
    q = torch.zeros(3, 2, 64, device=dev, dtype=BF)
    table, pos = qlinear.rope_table(64, 10), torch.zeros(3, dtype=torch.int64, device=dev)
    kc = torch.zeros(2, 2, 16, 64, device=dev, dtype=BF)
    for bad in (dict(q=q[0]), dict(k=q[:2]), dict(table=table.double()), dict(pos=pos.int()), dict(pos=pos[:2]), dict(layout="other"),
                dict(k=q.half()), dict(pos=pos.cpu())):
        a = dict(q=q, k=q, table=table, pos=pos, layout="half")
        a.update(bad)
        with pytest.raises((ValueError, TypeError)):
            qlinear.rope(a["q"], a["k"], a["table"], a["pos"], layout=a["layout"])
    with pytest.raises(qlinear.QlError):  # the table is wider than the head
        qlinear.rope(q, q, qlinear.rope_table(128, 10), pos)
    for kcache, slots in ((kc.float(), pos), (kc[:, :1], pos), (kc.transpose(2, 3), pos), (kc[..., :32], pos), (kc, pos.int())):
        with pytest.raises((ValueError, TypeError)):
            qlinear.rope_append(q, q, q, table, pos, kcache, kcache, slots)
    bad_page = torch.zeros(2, 2, 12, 64, device=dev, dtype=BF)
    with pytest.raises(qlinear.QlError):
        qlinear.rope_append(q, q, q, table, pos, bad_page, bad_page, pos)


# ------------------------------------------------------------------------ paged attention

def paged(g, q_lens, kv_lens, Hq, Hkv, D, ps, dtype, spare=3, std=1.0):
    """Random caches with the sequences' pages in shuffled order; every place that no sequence
    owns (spare pages, the unused tail of each last page, table entries past the end) is poisoned."""
    per = [-(-n // ps) for n in kv_lens]
    P = sum(per) + spare
    kc, vc = rnd(g, P, Hkv, ps, D, dtype=dtype, std=std), rnd(g, P, Hkv, ps, D, dtype=dtype)
    order = torch.randperm(P, generator=g, device="cuda").cpu()
    table = torch.full((len(kv_lens), max(per + [1]) + 1), -12345, dtype=torch.int32)
    at = 0
    used = torch.zeros(P, ps, dtype=torch.bool)
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n].int()
        for j in range(n):
            used[order[at + j], :min(ps, kv_lens[i] - j * ps)] = True
        at += n
    stale = ~used.cuda()
    kc.transpose(1, 2)[stale] = math.nan
    vc.transpose(1, 2)[stale] = math.inf
    starts = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
    q = rnd(g, sum(q_lens), Hq, D, dtype=dtype)
    return q, kc, vc, table.cuda(), starts, torch.tensor(kv_lens, dtype=torch.int32, device="cuda")


def attention_reference(q, kc, vc, table, q_lens, kv_lens, scale, causal, window):
    """(o, softmax @ |v|) in 64 bits."""
    T, Hq, D = q.shape
    Hkv, ps = kc.shape[1], kc.shape[2]
    G = Hq // Hkv
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    at = 0
    for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
        if n and L:
            pages = table[b, :-(-L // ps)].long()
            k = kc[pages].transpose(1, 2).reshape(-1, Hkv, D)[:L].double().repeat_interleave(G, 1)
            v = vc[pages].transpose(1, 2).reshape(-1, Hkv, D)[:L].double().repeat_interleave(G, 1)
            s = torch.einsum("ihd,jhd->hij", q[at:at + n].double(), k) * scale
            j, i = torch.arange(L, device=q.device), torch.arange(n, device=q.device)[:, None] + (L - n)
            see = (j <= i) if causal else torch.ones(n, L, dtype=torch.bool, device=q.device)
            if window:
                see = see & (j > i - window)
            p = torch.softmax(s.masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
            o[at:at + n] = torch.einsum("hij,jhd->ihd", p, v)
            a[at:at + n] = torch.einsum("hij,jhd->ihd", p, v.abs())
        at += n
    return o, a


def check_attention(g, q_lens, kv_lens, Hq, Hkv, D, ps=16, dtype=BF, causal=True, window=0, scale=None, std=1.0, view=None,
                    max_q=None, max_kv=None):
    q, kc, vc, table, starts, lens = paged(g, q_lens, kv_lens, Hq, Hkv, D, ps, dtype, std=std)
    if view is not None:
        q = view(q)
    got = qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=max_q or max(q_lens), max_kv=max_kv or max(kv_lens), scale=scale,
                                  causal=causal, window=window)
    o, a = attention_reference(q, kc, vc, table, q_lens, kv_lens, scale or D ** -0.5, causal, window)
    assert got.dtype == dtype and got.is_contiguous()
    # weights rounded to the dtype (u), the output rounded (u); fp32 scores: |q||k| sums of D
    # products, relative 2^-24 each, become absolute errors of the exponent (bounded by 64 * 2^-24
    # of the largest exponent, here below 2^7 * std); f16 weights under 2^-14 lose bits (2^-25 each)
    e = 2.0 ** -24 * 64 * 2 ** 7 * std
    low = max(kv_lens) * 2.0 ** -25 * 8 if dtype == HF else 0.0
    within(got, o, U[dtype] * (a + o.abs()) + 2 * e * a + low, "o")
    assert qlinear.device_error() == 0
    return got


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,Hkv", [(24, 8), (4, 4), (5, 1), (16, 2)])
def test_attention_single_tokens(D, dtype, Hq, Hkv):
    kv = [1, 2, 15, 16, 17, 127, 128, 129, 700]
    check_attention(gen(D + Hq), [1] * len(kv), kv, Hq, Hkv, D, 16, dtype)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("ps", [16, 32, 128, 256, 1024])
def test_attention_chunks_of_every_page_size(D, ps):
    check_attention(gen(D + ps), [5, 1, 130, 64], [300, 1, 130, 1100], 6, 2, D, ps)


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 24, 8), (64, 8, 8), (128, 7, 1), (128, 40, 2), (64, 3, 1)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 37), (True, 128), (True, 100000)])
def test_attention_masks(D, Hq, Hkv, dtype, causal, window):
    """Lengths around the tiles' edges; sequences without new tokens and without anything cached."""
    q = [1, 17, 128, 0, 200, 85, 86, 3, 257]
    kv = [512, 17, 129, 50, 200, 86, 600, 400, 385]
    check_attention(gen(D + window), q, kv, Hq, Hkv, D, 32, dtype, causal, window)


def test_attention_rows_that_see_nothing():
    """kv_len 0, and more new tokens than cached positions: those tokens get zeros."""
    for D in (64, 128):
        g = gen(D)
        got = check_attention(g, [3, 5, 40, 4], [0, 2, 9, 4], 6, 2, D)
        assert not got[:3].any() and not got[3:6].any() and got[6:8].any()
        check_attention(g, [3, 300], [0, 200], 6, 2, D)
        check_attention(g, [2, 2], [0, 0], 6, 2, D, max_kv=1)
        check_attention(g, [300], [250], 6, 2, D, causal=False)


@pytest.mark.parametrize("q_len", [1, 2, 150])
def test_attention_long_contexts(q_len):
    check_attention(gen(q_len), [q_len, q_len], [20011, 33], 6, 2, 128, 64) if q_len < 33 else check_attention(
        gen(q_len), [q_len, q_len], [20011, 1000], 6, 2, 128, 64)


@pytest.mark.parametrize("q_len", [1, 140])
def test_attention_extreme_scores(q_len):
    """One score far above the rest, scores near the fp32 exponent's ends, equal scores."""
    g = gen(q_len)
    for std, scale in ((8.0, None), (1.0, 1e-6), (1.0, 3.0)):
        q, kc, vc, table, starts, lens = paged(g, [q_len], [700], 4, 2, 128, 16, BF, std=std)
        got = qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=q_len, max_kv=700, scale=scale)
        sc = scale or 128 ** -0.5
        o, a = attention_reference(q, kc, vc, table, [q_len], [700], sc, True, 0)
        # fp32 scores of size up to 128 * 5 * 5 * std * scale: their rounding moves the exponent
        e = 2.0 ** -24 * 128 * 25 * std * sc * 2
        within(got, o, U[BF] * (a + o.abs()) + 2 * e * a)


def test_attention_strides_and_pool_views():
    g = gen(1)
    fused = lambda q: torch.cat([q, rnd(g, q.shape[0], 4, q.shape[2])], 1)[:, :q.shape[1]]  # noqa: E731
    check_attention(g, [1, 40], [90, 77], 6, 2, 128, view=fused)
    heads_first = lambda q: q.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    check_attention(g, [1, 40], [90, 77], 6, 2, 128, view=heads_first)
    check_attention(g, [1], [90], 6, 2, 64, view=heads_first)
    shifted = lambda q: torch.cat([q.flatten()[:3], q.flatten()])[3:].view(q.shape)  # noqa: E731  (off the 16-byte grid)
    check_attention(g, [3], [90], 6, 2, 64, view=shifted)
    # a layer's caches as planes of one pool, page stride larger than a page
    q, kc, vc, table, starts, lens = paged(g, [2, 60], [90, 300], 6, 2, 128, 16, BF)
    wide = torch.stack([kc, vc], 1)
    a = qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=60, max_kv=300)
    b = qlinear.paged_attention(q, wide[:, 0], wide[:, 1], table, starts, lens, max_q=60, max_kv=300)
    assert torch.equal(a, b)
    # rows of a wider table
    big = torch.full((2, 99), -1, dtype=torch.int32, device="cuda")
    big[:, :table.shape[1]] = table
    c = qlinear.paged_attention(q, kc, vc, big[:, :table.shape[1]], starts, lens, max_q=60, max_kv=300)
    assert torch.equal(a, c)


def test_attention_offsets_past_32_bits():
    """Pages whose element offset exceeds 2^31 (and byte offset 2^32)."""
    P, Hkv, ps, D = 135_000, 8, 16, 128
    cache = torch.empty(P, Hkv, ps, D, dtype=BF, device="cuda")
    g = gen(2)
    pages = torch.tensor([P - 1, 3, P - 70, 131_072], dtype=torch.int32, device="cuda")
    cache[pages.long()] = rnd(g, 4, Hkv, ps, D)
    for n in (1, 60):
        q = rnd(g, n, 8, D)
        starts, lens = torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.tensor([61], dtype=torch.int32, device="cuda")
        got = qlinear.paged_attention(q, cache, cache, pages[None], starts, lens, max_q=n, max_kv=61)
        small = cache[pages.long()]
        o, a = attention_reference(q, small, small, torch.arange(4, device="cuda")[None], [n], [61], D ** -0.5, True, 0)
        within(got, o, U[BF] * (a + o.abs()) + 1e-3 * a)


@pytest.mark.parametrize("q_lens", [[1] * 5, [1, 70, 1, 200, 3]])
def test_attention_same_answer_on_any_stream_and_in_a_graph(q_lens):
    g = gen(4)
    kv = [a + b for a, b in zip(q_lens, [300, 5, 2000, 0, 77])]
    q, kc, vc, table, starts, lens = paged(g, q_lens, kv, 6, 2, 128, 16, BF)
    call = lambda: qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=max(q_lens), max_kv=4096)  # noqa: E731
    table = torch.nn.functional.pad(table, (0, 4096 // 16 - table.shape[1]), value=-1)
    first = call()
    assert torch.equal(first, call())  # nothing depends on the order in which work finishes
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
    # a replay reads the lengths of its time
    lens -= torch.tensor([100, 0, 700, 0, 1], dtype=torch.int32, device="cuda")
    graph.replay()
    shorter = [n - d for n, d in zip(kv, [100, 0, 700, 0, 1])]
    o, a = attention_reference(q, kc.nan_to_num(0, 0, 0), vc.nan_to_num(0, 0, 0), table, q_lens, shorter, 128 ** -0.5, True, 0)
    within(out, o, U[BF] * (a + o.abs()) + 1e-3 * a)
    assert qlinear.device_error() == 0


def test_attention_reports_bad_sizes_and_pages():
    g = gen(6)
    for n in (1, 64):
        q, kc, vc, table, starts, lens = paged(g, [n], [100], 4, 2, 64, 16, BF)
        assert qlinear.device_error() == 0
        bad = table.clone()
        bad[0, 2] = kc.shape[0]  # past the cache: reported, read as page 0
        qlinear.paged_attention(q, kc, vc, bad, starts, lens, max_q=n, max_kv=100)
        assert qlinear.device_error() == _lib.DEV_ERR_BAD_INDEX
        qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=n, max_kv=99)  # longer than promised
        assert qlinear.device_error() == _lib.DEV_ERR_BAD_INDEX
        qlinear.paged_attention(q, kc, vc, table, starts + 1, lens, max_q=n, max_kv=100)  # past q's tokens
        assert qlinear.device_error() == _lib.DEV_ERR_BAD_INDEX


def test_attention_refusals(dev):
    g = gen(7)
    q, kc, vc, table, starts, lens = paged(g, [1, 2], [10, 20], 4, 2, 64, 16, BF)
    ok = dict(q=q, k=kc, v=vc, t=table, s=starts, n=lens, max_q=2, max_kv=20)

    def call(**kw):
        a = dict(ok)
        a.update({k: v for k, v in kw.items() if k in a})
        rest = {k: v for k, v in kw.items() if k not in ok}
        return qlinear.paged_attention(a["q"], a["k"], a["v"], a["t"], a["s"], a["n"], max_q=a["max_q"], max_kv=a["max_kv"], **rest)

    call()
    for bad in (dict(q=q[0]), dict(q=q.half()), dict(k=kc[:, :1]), dict(t=table.long()), dict(t=table[:1]), dict(s=starts[:2]),
                dict(n=lens.long()), dict(t=table[:, :1]), dict(max_kv=10 ** 6), dict(n=lens.cpu()), dict(k=kc[..., :32], v=vc[..., :32]),
                dict(out=torch.empty(3, 4, 32, device=dev, dtype=BF))):
        with pytest.raises((ValueError, TypeError)):
            call(**bad)
    for bad in (dict(max_q=4), dict(max_q=-1), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(window=-1),
                dict(window=4, causal=False), dict(q=torch.cat([q, q[:, :1]], 1))):
        with pytest.raises(qlinear.QlError):
            call(**bad)
    small = torch.zeros(4, 2, 8, 64, device=dev, dtype=BF)
    with pytest.raises(qlinear.QlError):  # page size
        call(k=small, v=small)
    odd = torch.zeros(4, 2, 16, 72, device=dev, dtype=BF)
    with pytest.raises(qlinear.QlError):  # head dimension
        call(q=torch.zeros(3, 4, 72, device=dev, dtype=BF), k=odd, v=odd)
    with pytest.raises(qlinear.QlError):
        call(q=q.float(), k=kc.float(), v=vc.float())


@pytest.mark.parametrize("q_len,kv", [(200, 1500), (30, 100)])
def test_attention_wait_runs_out_and_reports(q_len, kv):
    """With a loader that issues nothing (a flag that only this sets) and the wait limit at 50 ms,
    the launch ends by itself, the timeout is reported, and the next call is right."""
    g = gen(9)
    q, kc, vc, table, starts, lens = paged(g, [q_len], [kv], 6, 2, 128, 16, BF)
    assert qlinear.device_error() == 0
    try:
        _lib.debug_inject(_lib.INJECT_ATTENTION_PRODUCER_SILENT, 50_000_000)
        qlinear.paged_attention(q, kc, vc, table, starts, lens, max_q=q_len, max_kv=kv)
        err = qlinear.device_error()
    finally:
        _lib.debug_inject(0, 0)
    assert err & (_lib.DEV_ERR_TIMEOUT_FULL | _lib.DEV_ERR_TIMEOUT_EMPTY | _lib.DEV_ERR_TIMEOUT_ACC)
    check_attention(gen(10), [q_len], [kv], 6, 2, 128)


# ------------------------------------------------------------------------ pages

@pytest.mark.parametrize("shape", [(9, 2, 16, 64), (3, 2, 40, 1, 16, 8), (1, 12, 3, 128, 256), (70000, 3, 1, 8, 1)])
@pytest.mark.parametrize("dtype", [BF, F32, torch.uint8])
def test_copy_pages(shape, dtype):
    if shape[-1] == 1:
        shape = shape[:-1] + (16 // dtype.itemsize,)  # many planes of one 128-byte page
    g = gen(len(shape))
    pool = torch.randint(0, 255, shape, generator=g, device="cuda").to(dtype)
    P = shape[-4]
    order = torch.randperm(P, generator=g, device="cuda").tolist()
    n = P // 2
    want = pool.clone()
    want.select(-4, 0)  # pages are axis -4
    idx = [slice(None)] * (len(shape) - 4)
    want[tuple(idx + [order[n:2 * n]])] = pool[tuple(idx + [order[:n]])]
    qlinear.copy_pages(pool, order[:n], order[n:2 * n])
    assert torch.equal(pool, want)
    qlinear.copy_pages(pool, [], [])
    assert torch.equal(pool, want)


def test_copy_pages_of_a_long_list_and_one_source_many_times():
    pool = torch.arange(3000, device="cuda", dtype=torch.int32)[:, None, None, None].expand(3000, 1, 2, 4).contiguous()
    qlinear.copy_pages(pool, [7] * 1100, list(range(100, 1200)))
    assert (pool[100:1200] == 7).all() and torch.equal(pool[1200:, 0, 0, 0], torch.arange(1200, 3000, device="cuda", dtype=torch.int32))


def test_copy_pages_refusals(dev):
    pool = torch.zeros(8, 2, 16, 64, device=dev, dtype=BF)
    for src, dst in (([0], [8]), ([-1], [2]), ([8], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [0]), ([0], [-1])):
        with pytest.raises(qlinear.QlError):
            qlinear.copy_pages(pool, src, dst)
    with pytest.raises(ValueError):
        qlinear.copy_pages(pool, [0, 1], [2])
    with pytest.raises(ValueError):
        qlinear.copy_pages(pool, [1 << 40], [2])
    with pytest.raises(ValueError):
        qlinear.copy_pages(pool.transpose(0, 1), [0], [1])
    with pytest.raises(ValueError):
        qlinear.copy_pages(pool.cpu(), [0], [1])
    with pytest.raises(qlinear.QlError):  # a page of 2 bytes
        qlinear.copy_pages(torch.zeros(4, 1, 1, 1, device=dev, dtype=BF), [0], [1])
    assert not pool.any()
