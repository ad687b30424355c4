"""Activations kept in 8 bits.

``save8`` turns a tensor into int8 codes with a power-of-two scale for every
block of 32 values along the last dim (the last block of a row may be shorter),
8.25 bits a value instead of 16 or 32; ``load8`` gives the values back.  A
training layer that keeps its input this way holds half the memory until its
backward pass (``ops.dense.mixed_linear`` / ``mixed_ffn`` with ``save8=True``).

A block's scale is the smallest power of two with ``max |x| <= 127 * scale`` (at
least 2^-126), a code the integer nearest to ``x / scale``: values come back
within half a scale, at most 1/127 of the block's largest magnitude (2^-127 in
blocks at the smallest scale).  At the type's largest values codes are held to
63, so that nothing loads as an infinity: the top step is off by up to a whole
scale.  A code times its scale has 7 significant bits, so values are exact in
bf16.  A block that holds a NaN or an infinity loads as NaN.

Native path: ``_int8`` kernels (bf16, fp16 or fp32).  Eager path (CPU tensors,
or ``PD_KERNELS=eager``): the same bits in PyTorch.
"""
from __future__ import annotations

import os

import torch
from torch.autograd import forward_ad

from primus_dlrm_b200.ops import _ext

BLOCK = 32
_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_NAN = 255                        # scale byte of a block without numbers


class Saved8:
    """A tensor in 8 bits: ``codes`` int8 of its shape, ``exponents`` uint8
    ``[..., blocks]`` (the scale of byte ``e`` is ``2^(e - 127)``; 255: the block
    loads as NaN), and the ``shape`` and ``dtype`` that it had."""

    def __init__(self, codes: torch.Tensor, scale_bytes: torch.Tensor, shape, dtype: torch.dtype):
        # [rows, K] and block-major [blocks, rows]: a GEMM epilogue's threads own rows
        self._codes, self._bytes, self.shape, self.dtype = codes, scale_bytes, shape, dtype

    @property
    def codes(self) -> torch.Tensor:
        return self._codes.view(self.shape)

    @property
    def exponents(self) -> torch.Tensor:
        return self._bytes.t().unflatten(0, self.shape[:-1]) if len(self.shape) > 1 else self._bytes[:, 0]

    @property
    def nbytes(self) -> int:
        return self._codes.numel() + self._bytes.numel()


def _native(t: torch.Tensor) -> bool:
    return t.is_cuda and os.environ.get("PD_KERNELS") != "eager"


def no_tangent(who: str, *tensors: torch.Tensor | None) -> None:
    """Forward-mode derivatives do not pass through codes: refused, not dropped."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{who} has no forward-mode derivative")


def _save_ref(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    rows, K = x.shape
    blocks = -(-K // BLOCK)
    top = 137 if x.dtype == torch.float16 else 249           # where code 64 would pass the type's largest value
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - K)).view(rows, blocks, BLOCK)
    bits = x.abs().amax(-1).view(torch.int32)                # torch's maximum keeps a NaN
    byte = torch.where(bits >= 0x7F800000, _NAN, (((bits + 0x1FFFF) >> 23) - 6).clamp(min=1))
    inv = torch.where(byte == _NAN, 0, (254 - byte) << 23).int().view(torch.float32)
    most = torch.where(byte == _NAN, 0.0, torch.where(byte == top, 63.0, 127.0))[..., None]
    codes = torch.round(torch.nan_to_num(x * inv[..., None])).clamp(-most, most).to(torch.int8)
    return codes.view(rows, blocks * BLOCK)[:, :K].contiguous(), byte.to(torch.uint8).t().contiguous()


def _load_ref(codes: torch.Tensor, scale_bytes: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    byte = scale_bytes.t().int()
    scale = torch.where(byte == _NAN, torch.nan, (byte << 23).view(torch.float32))
    return (codes.float() * scale.repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]).to(dtype)


def save_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes [rows, K], scale bytes [blocks, rows]) of x [rows, K]."""
    return tuple(_ext.int8().save8(x)) if _native(x) else _save_ref(x)


def load_rows(codes: torch.Tensor, scale_bytes: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The values [rows, K] of :func:`save_rows`."""
    return _ext.int8().load8(codes, scale_bytes, dtype) if _native(codes) else _load_ref(codes, scale_bytes, dtype)


def save8(x: torch.Tensor) -> Saved8:
    """``x`` ``[..., K]`` (bf16, fp16 or fp32, any strides) in 8 bits.  Not
    differentiable: the result carries no graph."""
    if x.dim() == 0 or x.dtype not in _TYPES:
        raise ValueError(f"save8: a bf16, fp16 or fp32 tensor with a last dim is expected, not {x.dtype} of {x.dim()} dims")
    if _native(x):
        codes, scale_bytes = _ext.int8().save8(x)
    else:
        no_tangent("save8", x)
        codes, scale_bytes = _save_ref(x.detach().reshape(x.shape[:-1].numel(), x.shape[-1]))
    return Saved8(codes, scale_bytes, x.shape, x.dtype)


def load8(saved: Saved8, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values of a :class:`Saved8`, in the type that they had or in ``dtype``."""
    dtype = saved.dtype if dtype is None else dtype
    if dtype not in _TYPES:
        raise ValueError(f"load8: {dtype}: expected bf16, fp16 or fp32")
    return load_rows(saved._codes, saved._bytes, dtype).view(saved.shape)
