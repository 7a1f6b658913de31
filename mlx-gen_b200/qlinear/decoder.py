"""Decoder operators: what stands between the quantized linears of a decoder layer or a DiT
block -- the residual norm, rotary positions with the append to a paged cache, attention over
that cache (with a window and sinks), copies of its pages -- and between one decode step and the next:
sampling and the next step's index tensors.

torch holds the device memory and names the stream; the arithmetic runs in libqlinear's
kernels (include/qlinear.h describes each call).  Wrong shapes, types and devices raise
ValueError or TypeError here; a QlError comes from the library's own checks.
"""
from __future__ import annotations

import ctypes
import math
import os
import re
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import ROPE_HALF, ROPE_INTERLEAVED, lib

_LAYOUTS = {"half": ROPE_HALF, "interleaved": ROPE_INTERLEAVED}


class _Native:
    """qlinear._native (csrc/native.cpp), loaded and given libqlinear's functions on first use."""

    def __getattr__(self, name):
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_native.so")
        if not os.path.exists(path):
            raise ImportError(f"{path} not found; build it first (python -c 'import __graft_entry__ as g; g.build()')")
        from . import _native as m
        if not re.match(re.escape(m.torch_version) + r"(?!\d)", torch.__version__):  # its tensors are that torch's
            raise ImportError(f"{path} was built for torch {m.torch_version}, this is {torch.__version__}; build it again")
        L = lib()
        m.init(_lib.QlError, *(ctypes.cast(getattr(L, f), ctypes.c_void_p).value for f in (
            "ql_last_error", "ql_norm_residual", "ql_rope", "ql_rope_append", "ql_paged_attention",
            "ql_paged_attention_workspace_size", "ql_copy_pages", "ql_sink_attention", "ql_plan_step_within", "ql_sample")))
        for f in ("norm_residual", "rope", "rope_append", "paged_attention", "copy_pages", "plan_step", "sample"):
            setattr(self, f, getattr(m, f))
        return self.__dict__[name]


_native = _Native()


def _layout(name: str) -> int:
    if name not in _LAYOUTS:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {name!r}")
    return _LAYOUTS[name]


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
    return _native.norm_residual(y, residual, weight, post_weight, gate, gate_period, alpha, scale, scale_period, eps,
                                 weight_offset)


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


def rope(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, *,
         layout: str = "half") -> Tuple[torch.Tensor, torch.Tensor]:
    """Rotary positions on q ``[T, Hq, D]`` and k ``[T, Hk, D]`` (views with any token and head
    stride); returns new contiguous tensors.  The table's width is the rotary dimension (the rest
    of each head is copied); ``positions [T]`` (int64) are its rows.  layout "half" pairs (i, i +
    rotary_dim / 2), "interleaved" (2i, 2i + 1)."""
    return _native.rope(q, k, table, positions, _layout(layout))


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, positions: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *,
                layout: str = "half") -> torch.Tensor:
    """``rope`` with the rotated k and v written to the paged cache ``[pages, Hkv, page_size, D]`` at
    ``slots [T]`` (int64, page * page_size + offset; negative: not cached); returns the rotated q."""
    return _native.rope_append(q, k, v, table, positions, k_cache, v_cache, slots, _layout(layout))


# ------------------------------------------------------------------------ paged attention

def paged_attention_workspace_size(T: int, Hq: int, Hkv: int, D: int, B: int, max_q: int, max_kv: int,
                                   window: int = 0) -> int:
    """Bytes of workspace ``paged_attention`` needs for these sizes (0: none)."""
    return int(lib().ql_paged_attention_workspace_size(T, Hq, Hkv, D, B, max_q, max_kv, window))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    q_starts: torch.Tensor, kv_lens: torch.Tensor, *, max_q: int, max_kv: int,
                    scale: Optional[float] = None, causal: bool = True, window: int = 0, sinks: int = 0,
                    out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of each sequence's new tokens over its pages (their own keys and values already
    appended).  q ``[T, Hq, D]``: all sequences' new tokens, sequence b's from ``q_starts[b]`` to
    ``q_starts[b + 1]`` (int32 ``[B + 1]``); caches ``[pages, Hkv, page_size, D]``; ``page_table
    [B, n]`` and ``kv_lens [B]`` (new tokens included) int32.  max_q, max_kv: the longest chunk and
    the longest sequence (upper bounds are fine: a captured graph replays with the bounds it was
    captured with).  scale: ``1 / sqrt(D)`` by default.  Token i of q_len stands at ``p = kv_len -
    q_len + i`` and sees the positions up to p (all, without ``causal``), with a window only the
    last ``window`` of them and, with sinks (at most 1024), the sequence's first ``sinks`` positions, which
    stay visible; pages between the two are not used and may be given back.  Returns ``[T, Hq, D]``; a token that sees nothing gets zeros."""
    return _native.paged_attention(q, k_cache, v_cache, page_table, q_starts, kv_lens, max_q, max_kv, scale, causal, window,
                                   sinks, out, workspace)


# ------------------------------------------------------------------------ from step to step

def plan_step(page_table: torch.Tensor, lengths: torch.Tensor, new_tokens: torch.Tensor, *, page_size: int, max_tokens: int,
              max_kv: Optional[int] = None, free_pages: Optional[torch.Tensor] = None, taken: Optional[torch.Tensor] = None,
              out: Optional[tuple] = None) -> tuple:
    """The index tensors of a step in which sequence b, ``lengths[b]`` tokens long, gets ``new_tokens[b]``
    more (int32 ``[B]`` both): returns ``(positions, slots, q_starts, kv_lens, taken)`` for ``rope_append`` and
    ``paged_attention`` -- int64 ``[max_tokens]`` twice, int32 ``[B + 1]`` and ``[B]``; rows behind the last new token
    get position 0 and slot -1 (not cached).

    ``page_table [B, pages]`` (int32).  With a free list -- ``free_pages`` (int32) and ``taken [1]``, the number of its
    entries in use -- pages that the new tokens need are taken from it in the order of the sequences
    and entered in the page table; the returned ``taken`` counts them.  Without, the table holds every page
    already and ``taken`` is None.  A step that finds too few pages, columns or rows, or after which a sequence would
    hold more than ``max_kv`` tokens (or with counts below 0) has no tokens and changes nothing; ``device_error()`` tells.  ``out``: what an earlier call returned, to be
    written again; its kv_lens may be ``lengths`` and its taken ``taken``, so that each replay of a captured call
    goes one step on."""
    return _native.plan_step(page_table, lengths, new_tokens, page_size, max_tokens, max_kv, free_pages, taken, out)


MAX_SAMPLE_ROW = 1310208  # bytes of a row of logits that `sample` takes


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, logprobs: bool = False):
    """One token per row of ``logits [B, V]`` from the random numbers ``u [B]`` (float32 in [0, 1)): int64 ``[B]``,
    with ``logprobs`` also the logarithms of the probabilities with which they were drawn (float32 ``[B]``)::

        w_i = exp((x_i - max x) / temperature)
        in the order of x (descending, equal ones by index) stay: the first top_k; of those the shortest
        prefix with a sum of at least top_p times theirs; of those the ones with w_i >= min_p
        token = the first that stays, by index, with (sum up to it) > u * (sum of all that stay)

    Each setting is a number or a tensor ``[B]`` (float32, top_k int32) with each row's own; top_k 0, top_p 1 and
    min_p 0 filter nothing.  temperature 0 takes the largest logit, the lowest index of equal ones.
    Weights are summed exactly, as multiples of 2^-46 (to 2^-43, for more than 131072 tokens), so a row's token does not depend on the
    rest of the batch, and one whose weight rounds to 0 is never drawn (not by u = 0 either).  Logits of +inf share everything.  A row with a NaN
    (among the logits or its settings), a negative temperature or no logit above -inf gives token -1 and log-probability NaN."""
    return _native.sample(logits, u, temperature, top_k, top_p, min_p, logprobs)


# ------------------------------------------------------------------------ pages

def copy_pages(pool: torch.Tensor, src: Sequence[int], dst: Sequence[int]) -> None:
    """Page ``dst[i] := src[i]`` in every plane of a pool ``[..., pages, heads, page_size, head_dim]``
    (leading axes: layers, keys and values).  src and dst are host sequences; every page may be a
    destination once and no destination may be a source."""
    _native.copy_pages(pool, src, dst)
