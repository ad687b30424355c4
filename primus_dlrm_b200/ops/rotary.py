"""Norms of queries and keys for each head, with the position rotation.

``qk_norm_rope`` scales every head of every token to unit root mean square
(times a weight) and turns it by its position's angles, queries and keys in
one launch, forward and backward.  Rotated queries and keys depend on their
positions only through differences, so a model that uses it attends over
histories that grow, and over a key/value cache, without learned positions.

Native path: ``_kv.rotary`` (bf16, fp16 or fp32 in and out, 32-bit arithmetic,
its gradient node in C++).  Eager path: the same formulas in PyTorch.
"""
from __future__ import annotations

import os

import torch

from primus_dlrm_b200.ops import _ext

def _err_word(device) -> torch.Tensor:
    device = torch.device(device)
    return _ext.kv().rotary_err(torch.cuda.current_device() if device.index is None else device.index)


def rotary_error_code(device) -> int:
    """Error word of the rotary kernels (0 = ok, 1 = a position outside the
    angle table: its rows came out as zeros)."""
    return int(_err_word(device).item())


def rope_table(n_pos: int, rotary_dim: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """Angle table fp32 ``[n_pos, rotary_dim]``: the cosines of the
    ``rotary_dim / 2`` frequencies ``theta^(-2i / rotary_dim)`` at each
    position, then the sines (computed in 64 bits)."""
    if rotary_dim % 2 or rotary_dim < 0:
        raise ValueError(f"rotary_dim {rotary_dim}: expected an even number")
    inv = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / max(rotary_dim, 1))
    ang = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], dim=1).float()


def rotate_ref(x: torch.Tensor, angles: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """x ``[..., H, d]`` turned by ``angles`` ``[..., rotary_dim]`` (rows of a table)."""
    h = angles.shape[-1] // 2
    cos, sin = angles[..., None, :h].to(x.dtype), angles[..., None, h:].to(x.dtype)
    r, rest = x[..., :2 * h], x[..., 2 * h:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :h], r[..., h:])
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, rest], -1)


def _norm_rope_ref(x, weight, angles, eps, interleaved):
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    return rotate_ref(y, angles, interleaved).to(x.dtype)


def qk_norm_rope_ref(q, k, q_weight, k_weight, table, positions=None, eps: float = 1e-6, interleaved: bool = False):
    """Eager form of :func:`qk_norm_rope` (differentiable through autograd)."""
    T = (k if k is not None else q).shape[1]
    pos = torch.arange(T, device=q.device) if positions is None else positions.long()
    if pos.numel() and (int(pos.min()) < 0 or int(pos.max()) >= table.shape[0]):
        raise IndexError(f"a position lies outside the angle table of {table.shape[0]} rows")
    ang = table[pos]
    yq = _norm_rope_ref(q, q_weight, ang[..., T - q.shape[1]:, :], eps, interleaved)
    return yq, None if k is None else _norm_rope_ref(k, k_weight, ang, eps, interleaved)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor | None,
                 k_weight: torch.Tensor | None, table: torch.Tensor, positions: torch.Tensor | None = None, *,
                 eps: float = 1e-6, interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """RMS norm of each head, then the rotation by its position's angles.

    ``q`` ``[B, Tq, Hq, d]`` and ``k`` ``[B, T, Hk, d]`` (or None) are bf16,
    fp16 or fp32 views with any strides over tokens and heads, for instance
    slices of a fused projection; the queries belong to the LAST ``Tq`` of the
    ``T`` tokens.  ``q_weight`` / ``k_weight`` ``[d]`` may be None.  ``table``
    comes from :func:`rope_table`; its width is the part of a head that turns
    (the rest is only normed).  ``positions`` is ``[T]`` or ``[B, T]`` (int32
    or int64), by default ``0..T-1``.  ``interleaved`` pairs neighbours
    ``(2i, 2i + 1)`` instead of halves ``(i, i + rotary_dim / 2)``.

    Returns contiguous ``(q', k')`` of the inputs' type; differentiable once,
    backward, in ``q``, ``k`` and both weights (the native path refuses a table
    that requires a gradient, and forward-mode tangents).  A row whose position lies outside the
    table comes out as zeros and sets :func:`rotary_error_code` (IndexError on
    the eager path).
    """
    if q.is_cuda and os.environ.get("PD_KERNELS") != "eager":
        return _ext.kv().rotary(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k must be [B, T, H, d]")
    if k is not None and q.shape[1] > k.shape[1]:
        raise ValueError(f"more query tokens ({q.shape[1]}) than key tokens ({k.shape[1]})")
    return qk_norm_rope_ref(q, k, q_weight, k_weight, table, positions, eps, interleaved)
