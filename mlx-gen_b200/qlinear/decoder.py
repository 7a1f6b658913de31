"""Decoder operators: what stands between the quantized linears of a decoder layer or a DiT
block -- the residual norm, rotary positions with the append to a paged cache, attention over
that cache, and copies of its pages.

torch holds the device memory and names the stream; the arithmetic runs in libqlinear's
kernels (include/qlinear.h describes each call).  Wrong shapes, types and devices raise
ValueError or TypeError here; a QlError comes from the library's own checks.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import ROPE_HALF, ROPE_INTERLEAVED, check, lib

_DT = {torch.float32: _lib.QL_F32, torch.bfloat16: _lib.QL_BF16, torch.float16: _lib.QL_F16}
_LAYOUTS = {"half": ROPE_HALF, "interleaved": ROPE_INTERLEAVED}


def _dtype(t: torch.Tensor) -> int:
    code = _DT.get(t.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float32, bfloat16 or float16")
    return code


def _call(device: torch.device, fn, *args) -> None:
    """One library call on `device`'s current stream."""
    i = device.index
    if i != torch.cuda.current_device():
        with torch.cuda.device(i):
            check(fn(*args, torch._C._cuda_getCurrentRawStream(i)))
    else:
        check(fn(*args, torch._C._cuda_getCurrentRawStream(i)))


def _on(device: torch.device, **tensors: Optional[torch.Tensor]) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


def _cuda(t: torch.Tensor) -> torch.device:
    if not t.is_cuda:
        raise ValueError("libqlinear operates on CUDA tensors only")
    return t.device


def _row(name: str, t: Optional[torch.Tensor], like: torch.Tensor, D: int, rows: int = 1) -> int:
    """Pointer of a contiguous [rows.., D] operand in `like`'s dtype (0: absent)."""
    if t is None:
        return 0
    if t.dtype != like.dtype or t.device != like.device:
        raise TypeError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    if t.shape[-1] != D or t.numel() < rows * D:
        raise ValueError(f"{name} must hold {rows} row(s) of {D} elements, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


# ------------------------------------------------------------------------ residual norm

def norm_residual(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *,
                  post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, gate_period: int = 0,
                  alpha: float = 1.0, scale: Optional[torch.Tensor] = None, scale_period: int = 0, eps: float = 1e-5,
                  weight_offset: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The norms around a block, fused with its gate and residual scale; returns ``(h, r)``::

        u = rms(y) * (weight_offset + post_weight)      # y itself without post_weight
        r = residual + alpha * gate * u                 # the residual stream after the block
        h = rms(r) * (weight_offset + weight) * (1 + scale)     # what the next block reads

    with ``rms(x) = x / sqrt(mean(x^2) + eps)`` over the last axis, in fp32 with one rounding per
    output.  y ``[..., D]``; residual of the same shape in y's dtype or float32; weights ``[D]``;
    gate / scale ``[D]`` or ``[rows, D]`` with row ``m // period`` for row m of y.  The DiT blocks'
    ``residual + gate * norm(branch)`` is post_weight and gate (src/nn.rs:166-176 for the gated
    sum); a decoder layer uses neither."""
    device = _cuda(y)
    D = y.shape[-1]
    if residual.shape != y.shape:
        raise ValueError(f"residual {tuple(residual.shape)} must have y's shape {tuple(y.shape)}")
    if residual.device != device:
        raise ValueError(f"residual is on {residual.device}, expected {device}")
    ydt, rdt = _dtype(y), _dtype(residual)
    M = y.numel() // D if D else 0
    y2 = y if y.dim() == 2 else y.reshape(-1, D)
    r2 = residual if residual.dim() == 2 else residual.reshape(-1, D)
    ys, rs = y2.stride(0), r2.stride(0)
    if y2.stride(1) != 1 or (M > 1 and ys < D):
        y2 = y2.contiguous()
        ys = D
    if r2.stride(1) != 1 or (M > 1 and rs < D):
        r2 = r2.contiguous()
        rs = D
    rows = lambda period: -(-M // period) if period > 0 else 1  # noqa: E731
    h = torch.empty(y.shape, dtype=y.dtype, device=device)
    r = torch.empty(y.shape, dtype=residual.dtype, device=device)
    _call(device, lib().ql_norm_residual, y2.data_ptr(), ydt, max(ys, D), r2.data_ptr(), rdt, max(rs, D), M, D,
          _row("weight", weight, y, D), weight_offset, _row("post_weight", post_weight, y, D),
          _row("gate", gate, y, D, rows(gate_period)), gate_period, alpha,
          _row("scale", scale, y, D, rows(scale_period)), scale_period, eps, h.data_ptr(), r.data_ptr())
    return h, r


# ------------------------------------------------------------------------ rotary positions

def rope_table(rotary_dim: int, positions, base: float = 10000.0, scaling: Optional[dict] = None,
               device="cuda") -> torch.Tensor:
    """Table of ``rope`` / ``rope_append``: float32 ``[P, rotary_dim]``, row p the cosines, then the
    sines, of position p's angles, computed in float64.

    positions: the number of positions, or a tensor of them ``[P]`` (any real values).  A tensor
    ``[P, axes]`` with ``scaling={"axes": (d0, d1, ..)}`` gives each axis its own d elements of
    the head, as the image and video transformers' positions do.  scaling, for long contexts:

    - ``{"type": "linear", "factor": f}``: positions divided by f;
    - ``{"type": "ntk", "factor": f}``: base times ``f^(dim / (dim - 2))``;
    - ``{"type": "llama3", "factor", "low_freq_factor", "high_freq_factor", "original_positions"}``:
      wavelengths above ``original / low`` divided by the factor, below ``original / high`` kept,
      a linear blend between;
    - ``{"type": "yarn", "factor", "original_positions"[, "beta_fast", "beta_slow", "magnitude"]}``:
      a linear blend over the dimensions between ``beta_fast`` and ``beta_slow`` turns within the
      original context, cosines and sines times ``0.1 ln(factor) + 1`` unless given.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    scaling = dict(scaling or {})
    axes = scaling.pop("axes", None)
    kind = scaling.pop("type", None)
    if isinstance(positions, torch.Tensor):
        pos = positions.to(device="cpu", dtype=torch.float64)
    else:
        pos = torch.arange(int(positions), dtype=torch.float64)
    if axes is not None:
        if pos.dim() != 2 or pos.shape[1] != len(axes) or sum(axes) != rotary_dim or any(d < 2 or d % 2 for d in axes):
            raise ValueError("axes must be even, sum to rotary_dim, and match positions [P, axes]")
    elif pos.dim() != 1:
        raise ValueError("positions must be [P] without axes")

    def take(name, default=None):
        v = scaling.pop(name, default)
        if v is None:
            raise ValueError(f"scaling {kind!r} needs {name!r}")
        return float(v)

    factor = take("factor") if kind else 1.0
    magnitude = 1.0
    if kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs rotary_dim >= 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))

    def freqs(d):
        nonlocal magnitude
        f = base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        if kind in (None, "ntk"):
            return f
        if kind == "linear":
            return f / factor
        if kind == "llama3":
            original = take("original_positions")
            low, high = take("low_freq_factor"), take("high_freq_factor")
            turns = original * f / (2 * math.pi)  # turns within the original context
            keep = ((turns - low) / (high - low)).clamp(0, 1)
            return f * (keep + (1 - keep) / factor)
        if kind == "yarn":
            original = take("original_positions")
            fast, slow = take("beta_fast", 32.0), take("beta_slow", 1.0)
            magnitude = take("magnitude", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
            # index (in pairs) of the dimension that makes `turns` turns within the original context
            at = lambda turns: d * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), d - 1)
            ramp = ((torch.arange(d // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
            return f * ((1 - ramp) + ramp / factor)
        raise ValueError(f"unknown scaling type {kind!r}")

    if axes is None:
        angles = pos[:, None] * freqs(rotary_dim)
    else:
        if kind in ("llama3", "yarn"):
            raise ValueError("axes go with linear or ntk scaling only")
        angles = torch.cat([pos[:, i:i + 1] * freqs(d) for i, d in enumerate(axes)], 1)
    if scaling:
        raise ValueError(f"unknown scaling entries {sorted(scaling)}")
    return torch.cat([angles.cos() * magnitude, angles.sin() * magnitude], 1).float().to(device)


def _heads(name: str, x: torch.Tensor, T: int, D: int, like: torch.Tensor) -> torch.Tensor:
    if x.dim() != 3 or x.shape[0] != T or x.shape[2] != D:
        raise ValueError(f"{name} must be [{T}, heads, {D}], got {tuple(x.shape)}")
    if x.dtype != like.dtype or x.device != like.device:
        raise TypeError(f"{name} must be {like.dtype} on {like.device}, got {x.dtype} on {x.device}")
    return x if x.stride(2) == 1 else x.contiguous()


def _rope_args(q, table, positions, layout):
    device = _cuda(q)
    if q.dim() != 3:
        raise ValueError(f"q must be [tokens, heads, head_dim], got {tuple(q.shape)}")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError("table must be a contiguous float32 [positions, rotary_dim] (see rope_table)")
    if positions.dtype != torch.int64 or positions.shape != q.shape[:1] or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int64 [tokens]")
    _on(device, table=table, positions=positions)
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    return device, _LAYOUTS[layout]


def rope(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, *,
         layout: str = "half") -> Tuple[torch.Tensor, torch.Tensor]:
    """Rotary positions on q ``[T, Hq, D]`` and k ``[T, Hk, D]`` (views with any token and head
    stride); returns new contiguous tensors.  The table's width is the rotary dimension (the rest
    of each head is copied); ``positions [T]`` (int64) are its rows.  layout "half" pairs (i, i +
    rotary_dim / 2), "interleaved" (2i, 2i + 1)."""
    device, lay = _rope_args(q, table, positions, layout)
    T, Hq, D = q.shape
    q = _heads("q", q, T, D, q)
    k = _heads("k", k, T, D, q)
    Hk = k.shape[1]
    qo = torch.empty((T, Hq, D), dtype=q.dtype, device=device)
    ko = torch.empty((T, Hk, D), dtype=q.dtype, device=device)
    _call(device, lib().ql_rope, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
          _dtype(q), T, Hq, Hk, D, table.shape[1], lay, table.data_ptr(), table.shape[0], positions.data_ptr(),
          qo.data_ptr(), ko.data_ptr())
    return qo, ko


def _cache_shape(k_cache: torch.Tensor, v_cache: torch.Tensor, like: torch.Tensor):
    """(pages, heads, page size, head dim, page stride) of a layer's two caches."""
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dim() != 4 or c.dtype != like.dtype or c.device != like.device:
            raise ValueError(f"{name} must be [pages, heads, page_size, head_dim] in {like.dtype} on {like.device}, got "
                             f"{tuple(c.shape)} {c.dtype} on {c.device}")
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError("k_cache and v_cache must have the same shape and strides")
    P, H, ps, D = k_cache.shape
    sp, sh, st, sd = k_cache.stride()
    if sd != 1 or st != D or (H > 1 and sh != ps * D) or (P > 1 and sp < H * ps * D):
        raise ValueError("the [heads, page_size, head_dim] of a page must be contiguous")
    return P, H, ps, D, sp if P > 1 else H * ps * D


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, positions: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *,
                layout: str = "half") -> torch.Tensor:
    """``rope`` with the rotated k and v written to the paged cache ``[pages, Hkv, page_size, D]`` at
    ``slots [T]`` (int64, page * page_size + offset; negative: not cached); returns the rotated q."""
    device, lay = _rope_args(q, table, positions, layout)
    T, Hq, D = q.shape
    q = _heads("q", q, T, D, q)
    k, v = _heads("k", k, T, D, q), _heads("v", v, T, D, q)
    P, H, ps, cd, stride = _cache_shape(k_cache, v_cache, q)
    if k.shape[1] != H or v.shape[1] != H or cd != D:
        raise ValueError(f"k and v must have the cache's {H} heads of {cd}, got {tuple(k.shape)} and {tuple(v.shape)}")
    if slots.dtype != torch.int64 or slots.shape != positions.shape or not slots.is_contiguous() or slots.device != device:
        raise ValueError(f"slots must be a contiguous int64 [tokens] on {device}")
    qo = torch.empty((T, Hq, D), dtype=q.dtype, device=device)
    _call(device, lib().ql_rope_append, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
          v.data_ptr(), v.stride(0), v.stride(1), _dtype(q), T, Hq, H, D, table.shape[1], lay, table.data_ptr(),
          table.shape[0], positions.data_ptr(), slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), P, stride, ps,
          qo.data_ptr())
    return qo


# ------------------------------------------------------------------------ paged attention

def paged_attention_workspace_size(T: int, Hq: int, Hkv: int, D: int, B: int, max_q: int, max_kv: int) -> int:
    """Bytes of workspace ``paged_attention`` needs for these sizes (0: none)."""
    return int(lib().ql_paged_attention_workspace_size(T, Hq, Hkv, D, B, max_q, max_kv))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    q_starts: torch.Tensor, kv_lens: torch.Tensor, *, max_q: int, max_kv: int,
                    scale: Optional[float] = None, causal: bool = True, window: int = 0,
                    out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of each sequence's new tokens over its pages (their own keys and values already
    appended).  q ``[T, Hq, D]``: all sequences' new tokens, sequence b's from ``q_starts[b]`` to
    ``q_starts[b + 1]`` (int32 ``[B + 1]``); caches ``[pages, Hkv, page_size, D]``; ``page_table
    [B, n]`` and ``kv_lens [B]`` (new tokens included) int32.  max_q, max_kv: the longest chunk and
    the longest sequence (upper bounds are fine: a captured graph replays with the bounds it was
    captured with).  scale: ``1 / sqrt(D)`` by default.  Token i of q_len stands at ``p = kv_len -
    q_len + i`` and sees the positions up to p (all, without ``causal``), with a window only the
    last ``window`` of them.  Returns ``[T, Hq, D]``; a token that sees nothing gets zeros."""
    device = _cuda(q)
    if q.dim() != 3:
        raise ValueError(f"q must be [tokens, heads, head_dim], got {tuple(q.shape)}")
    T, Hq, D = q.shape
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    P, Hkv, ps, cd, stride = _cache_shape(k_cache, v_cache, q)
    if cd != D:
        raise ValueError(f"q's head dimension {D} differs from the cache's {cd}")
    B = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    if (B < 0 or page_table.dim() != 2 or page_table.shape[0] != B or q_starts.shape != (B + 1,)):
        raise ValueError("expected kv_lens [B], q_starts [B + 1] and page_table [B, pages], got "
                         f"{tuple(kv_lens.shape)}, {tuple(q_starts.shape)}, {tuple(page_table.shape)}")
    for name, t in (("page_table", page_table), ("q_starts", q_starts), ("kv_lens", kv_lens)):
        if t.dtype != torch.int32 or t.device != device or (t.numel() and t.stride(-1) != 1):
            raise ValueError(f"{name} must be int32 on {device} with a contiguous last axis")
    if page_table.shape[1] * ps < max_kv:
        raise ValueError(f"page_table's {page_table.shape[1]} pages of {ps} do not hold max_kv={max_kv} positions")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device or not out.is_contiguous():
        raise ValueError("out must be contiguous, of q's shape, dtype and device")
    L = lib()
    need = L.ql_paged_attention_workspace_size(T, Hq, Hkv, D, B, max_q, max_kv)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    _call(device, L.ql_paged_attention, q.data_ptr(), _dtype(q), q.stride(0), q.stride(1), T, Hq, Hkv, D,
          k_cache.data_ptr(), v_cache.data_ptr(), P, stride, ps, page_table.data_ptr(),
          page_table.stride(0) if B > 1 else page_table.shape[1], q_starts.data_ptr(), kv_lens.data_ptr(), B, max_q, max_kv,
          1.0 / math.sqrt(D) if scale is None else scale, causal, window, out.data_ptr(),
          workspace.data_ptr() if need else 0, need)
    return out


# ------------------------------------------------------------------------ pages

def copy_pages(pool: torch.Tensor, src: Sequence[int], dst: Sequence[int]) -> None:
    """Page ``dst[i] := src[i]`` in every plane of a pool ``[..., pages, heads, page_size, head_dim]``
    (leading axes: layers, keys and values).  src and dst are host sequences; every page may be a
    destination once and no destination may be a source."""
    device = _cuda(pool)
    if pool.dim() < 4 or not pool.is_contiguous():
        raise ValueError("pool must be a contiguous [.., pages, heads, page_size, head_dim]")
    n = len(src)
    if len(dst) != n:
        raise ValueError(f"{n} sources for {len(dst)} destinations")
    pages = pool.shape[-4]
    if any(not -0x80000000 <= i <= 0x7fffffff for x in (src, dst) for i in (min(x, default=0), max(x, default=0))):
        raise ValueError("page index out of range")
    arr = C.c_int32 * n
    page_bytes = pool.shape[-3] * pool.shape[-2] * pool.shape[-1] * pool.element_size()
    planes = pool.numel() * pool.element_size() // (pages * page_bytes) if pages and page_bytes else 0
    _call(device, lib().ql_copy_pages, pool.data_ptr(), planes, pages * page_bytes, pages, page_bytes, page_bytes,
          arr(*src), arr(*dst), n)
