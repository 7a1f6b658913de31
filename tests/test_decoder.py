"""CPU: the decoder operators' host side -- rotary tables, the library's own argument checks (no
GPU call is reached), refusals of CPU tensors."""
import ctypes as C
import math

import pytest
import torch

import qlinear
from qlinear import _lib


def angles(table):
    half = table.shape[1] // 2
    return torch.atan2(table[:, half:].double(), table[:, :half].double())


def same_angle(got, want):
    d = (got - want + math.pi) % (2 * math.pi) - math.pi
    # fp32 cosine and sine: 2^-25 each, as an angle
    assert float(d.abs().max()) < 1e-6


def test_rope_table_plain_and_far_positions():
    t = qlinear.rope_table(8, 5, device="cpu")
    f = 10000.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
    assert t.shape == (5, 8) and t.dtype == torch.float32
    same_angle(angles(t), torch.arange(5, dtype=torch.float64)[:, None] * f)
    far = torch.tensor([131071.0, 10_000_003.0], dtype=torch.float64)
    same_angle(angles(qlinear.rope_table(128, far, base=5e5, device="cpu")),
               far[:, None] * 5e5 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128))


def test_rope_table_scalings():
    pos = torch.tensor([1.0], dtype=torch.float64)
    f = 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    one = lambda **s: angles(qlinear.rope_table(64, pos, scaling=s, device="cpu"))[0]  # noqa: E731
    same_angle(one(type="linear", factor=4.0), f / 4)
    same_angle(one(type="ntk", factor=4.0), (1e4 * 4 ** (64 / 62)) ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64))
    got = one(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_positions=8192)
    wave = 2 * math.pi / f
    for i in range(32):
        w = float(wave[i])
        if w < 8192 / 4:
            want = float(f[i])
        elif w > 8192:
            want = float(f[i]) / 8
        else:
            s = (8192 / w - 1) / 3
            want = float(f[i]) * ((1 - s) / 8 + s)
        assert abs(float(got[i]) - want) < 1e-6
    y = qlinear.rope_table(64, pos, scaling=dict(type="yarn", factor=4.0, original_positions=4096), device="cpu").double()
    size = (y[:, :32].square() + y[:, 32:].square()).sqrt()
    assert float((size - (0.1 * math.log(4) + 1)).abs().max()) < 1e-6
    got = angles(y)[0]
    assert abs(float(got[0]) - float(f[0])) < 1e-6 and abs(float(got[-1]) - float(f[-1]) / 4) < 1e-6
    assert all(float(f[i]) / 4 - 1e-6 <= float(got[i]) <= float(f[i]) + 1e-6 for i in range(32))


def test_rope_table_axes():
    pos = torch.tensor([[3.0, 5.0, 7.0], [0.0, 1.0, 2.0]], dtype=torch.float64)
    t = qlinear.rope_table(16, pos, scaling={"axes": (4, 4, 8)}, device="cpu")
    want = torch.cat([pos[:, i:i + 1] * 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d) for i, d in enumerate((4, 4, 8))], 1)
    same_angle(angles(t), want)


@pytest.mark.parametrize("args,kw", [((7, 4), {}), ((0, 4), {}), ((8, 4), dict(scaling={"type": "other", "factor": 2})),
                                     ((8, 4), dict(scaling={"type": "linear"})),
                                     ((8, 4), dict(scaling={"type": "linear", "factor": 2, "extra": 1})),
                                     ((8, 4), dict(scaling={"axes": (4, 4)})), ((8, torch.zeros(2, 2)), {}),
                                     ((8, torch.zeros(2, 2)), dict(scaling={"axes": (4, 2)})),
                                     ((2, 4), dict(scaling={"type": "ntk", "factor": 2}))])
def test_rope_table_refusals(args, kw):
    with pytest.raises(ValueError):
        qlinear.rope_table(*args, device="cpu", **kw)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        qlinear.norm_residual(x, x, x[0, 0])
    with pytest.raises(ValueError):
        qlinear.rope(x, x, torch.zeros(4, 64), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        qlinear.paged_attention(x, x[None], x[None], i32[None], i32, i32[:2], max_q=1, max_kv=1)
    with pytest.raises(ValueError):
        qlinear.copy_pages(x[None], [0], [1])


def _attention(L, p=C.c_void_p(0x1000), **kw):
    a = dict(q=p, dt=1, ts=256, hs=64, T=4, Hq=4, Hkv=2, D=64, k=p, v=p, P=8, pst=2 * 16 * 64, ps=16, tab=p, tst=8, qs=p, kl=p, B=2,
             mq=2, mk=100, scale=0.125, causal=1, window=0, out=p, ws=None, wb=0)
    a.update(kw)
    return L.ql_paged_attention(*a.values(), None)


def test_library_checks_need_no_gpu():
    L, p = _lib.lib(), C.c_void_p(0x1000)
    bad = C.c_void_p(0x1001)
    norm = lambda **kw: L.ql_norm_residual(*{**dict(y=p, dt=1, ys=64, r=p, rdt=1, rs=64, M=2, D=64, w=p, o=0.0, post=None, gate=None, gp=0,  # noqa: E731
                                                    alpha=1.0, scale=None, sp=0, eps=1e-5, h=p, ro=p), **kw}.values(), None)
    assert norm(M=0) == 0
    assert norm(D=0) == _lib.QL_EINVAL_SHAPE and norm(D=32769, ys=32769, rs=32769) == _lib.QL_EINVAL_SHAPE
    assert norm(ys=63) == _lib.QL_EINVAL_SHAPE and norm(rs=63) == _lib.QL_EINVAL_SHAPE
    assert norm(rdt=2) == _lib.QL_EUNSUPPORTED and norm(dt=7) == _lib.QL_EUNSUPPORTED
    for k in ("y", "r", "w", "h", "ro"):
        assert norm(**{k: None}) == _lib.QL_EINVAL_ARG and norm(**{k: bad}) == _lib.QL_EINVAL_ARG
    assert norm(gp=-1) == _lib.QL_EINVAL_ARG and norm(post=bad) == _lib.QL_EINVAL_ARG

    rope = lambda **kw: L.ql_rope(*{**dict(q=p, qt=128, qh=64, k=p, kt=64, kh=64, dt=1, T=3, Hq=2, Hk=1, D=64, rot=64, lay=0, tab=p, P=9,  # noqa: E731
                                           pos=p, qo=p, ko=p), **kw}.values(), None)
    assert rope(T=0) == 0
    for kw in (dict(rot=63), dict(rot=0), dict(rot=66), dict(D=0), dict(D=1026, rot=2), dict(Hq=0, Hk=0), dict(P=-1), dict(T=-1)):
        assert rope(**kw) == _lib.QL_EINVAL_SHAPE, kw
    assert rope(dt=3) == _lib.QL_EUNSUPPORTED and rope(lay=2) == _lib.QL_EINVAL_ARG
    for k in ("q", "k", "tab", "pos", "qo", "ko"):
        assert rope(**{k: None}) == _lib.QL_EINVAL_ARG, k
    assert rope(q=bad) == _lib.QL_EINVAL_ARG and rope(tab=bad) == _lib.QL_EINVAL_ARG

    for kw, rc in ((dict(D=80), 2), (dict(Hq=5), 1), (dict(Hkv=0), 1), (dict(B=70000), 1), (dict(mq=5), 1), (dict(mk=-1), 1), (dict(dt=0), 2),
                   (dict(ps=8), 2), (dict(ps=24), 2), (dict(ps=2048), 2), (dict(P=0), 1), (dict(pst=2047), 1), (dict(tst=6), 1),
                   (dict(scale=0.0), 4), (dict(scale=-1.0), 4), (dict(scale=math.nan), 4), (dict(window=-1), 4), (dict(window=5, causal=0), 4),
                   (dict(q=None), 4), (dict(q=bad), 4), (dict(ts=255), 4), (dict(kl=None), 4),
                   (dict(mk=1 << 31, tst=1 << 30), 1), (dict(T=1 << 20, mq=1 << 20, Hq=128, Hkv=2), 2)):
        assert _attention(L, **kw) == rc, kw
    assert _attention(L, T=0, mq=0) == 0 and _attention(L, B=0) == 0
    need = L.ql_paged_attention_workspace_size(4, 4, 2, 64, 2, 2, 100000, 0)
    assert need > 0
    assert _attention(L, mk=100000, tst=6250, ws=p, wb=need - 1) == _lib.QL_EINVAL_ARG and b"workspace" in L.ql_last_error()
    assert L.ql_paged_attention_workspace_size(4, 4, 2, 80, 2, 2, 100000, 0) == 0

    copy = lambda src, dst, **kw: L.ql_copy_pages(*{**dict(pool=p, planes=1, ps=0, P=8, st=64, pb=64), **kw}.values(),  # noqa: E731
                                                  (C.c_int32 * len(src))(*src), (C.c_int32 * len(dst))(*dst), len(src), None)
    assert copy([], []) == 0 and copy([0], [1], planes=0) == 0
    assert copy([0], [8]) == _lib.QL_EINVAL_ARG and copy([0, 1], [1, 2]) == _lib.QL_EINVAL_ARG and copy([0, 1], [2, 2]) == _lib.QL_EINVAL_ARG
    assert copy([0], [1], pb=24, st=32) == _lib.QL_EINVAL_SHAPE and copy([0], [1], st=48) == _lib.QL_EINVAL_SHAPE
    assert copy([0], [1], planes=2, ps=448) == _lib.QL_EINVAL_SHAPE and copy([0], [1], pool=bad) == _lib.QL_EINVAL_ARG
