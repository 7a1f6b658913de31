"""CPU: what the library and the Python functions refuse before any launch (sampling, step planning, sinks)."""
import ctypes as C
import math

import pytest
import torch

import qlinear
from qlinear import _lib

P, BAD = C.c_void_p(0x1000), C.c_void_p(0x1001)


def test_cpu_tensors_are_refused():
    x, u, n = torch.zeros(2, 8), torch.zeros(2), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        qlinear.sample(x, u)
    with pytest.raises(ValueError):
        qlinear.plan_step(n.view(2, 1), n, n, page_size=16, max_tokens=1)
    with pytest.raises(TypeError):
        qlinear.sample(None, u)
    with pytest.raises(TypeError):
        qlinear.plan_step(n.view(2, 1), n, n, page_size=16)


def test_sample():
    call = lambda **kw: _lib.lib().ql_sample(*{**dict(x=P, dt=1, rs=100, B=2, V=100, u=P, t=None, ta=1.0, k=None, ka=0, p=None, pa=1.0,  # noqa: E731
                                                      m=None, ma=0.0, tok=P, lp=None), **kw}.values(), None)
    assert call(B=0) == 0 and call(B=0, x=None, u=None, tok=None) == 0
    for kw in (dict(B=-1), dict(V=0), dict(rs=-1)):
        assert call(**kw) == _lib.QL_EINVAL_SHAPE, kw
    for kw in (dict(dt=3), dict(V=655105, rs=655105), dict(V=327553, rs=327553, dt=0), dict(V=1 << 40)):
        assert call(**kw) == _lib.QL_EUNSUPPORTED, kw
    for kw in (dict(x=None), dict(u=None), dict(tok=None), dict(x=BAD), dict(u=BAD), dict(tok=C.c_void_p(0x1004)), dict(lp=BAD), dict(t=BAD),
               dict(k=BAD), dict(p=BAD), dict(m=BAD), dict(ta=-1.0), dict(ta=math.nan), dict(ka=-1), dict(pa=-0.5), dict(pa=math.nan),
               dict(ma=-0.1), dict(ma=1.1), dict(ma=math.nan)):
        assert call(**kw) == _lib.QL_EINVAL_ARG, kw
        assert _lib.lib().ql_last_error()


def test_plan_step():
    call = lambda **kw: _lib.lib().ql_plan_step(*{**dict(t=P, ts=8, tw=8, n=P, c=P, B=2, ps=16, T=4, f=P, nf=3, tk=P, pos=P, sl=P, qs=P, kv=P,  # noqa: E731
                                                         to=P), **kw}.values(), None)
    for kw in (dict(B=-1), dict(T=-1), dict(T=1 << 31), dict(nf=-1), dict(nf=1 << 31), dict(ts=7), dict(tw=-1), dict(B=(1 << 31) - 1)):
        assert call(**kw) == _lib.QL_EINVAL_SHAPE, kw
    for ps in (0, -16, 12, 24):
        assert call(ps=ps) == _lib.QL_EUNSUPPORTED
    for kw in (dict(t=None), dict(n=None), dict(c=None), dict(kv=None), dict(qs=None), dict(pos=None), dict(sl=None), dict(tk=None), dict(to=None),
               dict(t=BAD), dict(n=BAD), dict(c=BAD), dict(f=BAD), dict(tk=BAD), dict(pos=C.c_void_p(0x1004)), dict(sl=BAD), dict(qs=BAD), dict(kv=BAD)):
        assert call(**kw) == _lib.QL_EINVAL_ARG, kw


def test_sink_attention():
    base = dict(q=P, dt=1, ts=256, hs=64, T=4, Hq=4, Hkv=2, D=64, k=P, v=P, P=8, pst=2 * 16 * 64, ps=16, tab=P, tst=8, qs=P, kl=P, B=2, mq=2, mk=100,
                scale=0.125, window=20, sinks=4, out=P, ws=None, wb=0)
    call = lambda **kw: _lib.lib().ql_sink_attention(*{**base, **kw}.values(), None)  # noqa: E731
    assert call(T=0, mq=0) == 0 and call(B=0) == 0
    for kw in (dict(window=0), dict(sinks=-1), dict(window=-1), dict(q=None), dict(scale=0.0)):
        assert call(**kw) == _lib.QL_EINVAL_ARG, kw
    assert call(sinks=1025) == _lib.QL_EUNSUPPORTED and call(D=80) == _lib.QL_EUNSUPPORTED and call(mq=5) == _lib.QL_EINVAL_SHAPE
