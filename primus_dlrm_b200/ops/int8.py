"""Products of 8-bit integers, for serving.

A weight is laid out once as int8 codes with a 32-bit scale for each output
channel (:class:`Int8Weight`); every call turns its input's rows into codes with
a scale for each row, multiplies in integers (sums in 32 bits, exact) and applies
scales, bias, activation and residual in 32 bits:

    s_m = max(max_k |x_mk| * (1 / 127), 2^-126),  a_mk = rint(x_mk * (1 / s_m))
    y_mn = act((sum_k a_mk w_nk) * (s_m t_n) + bias_n) + residual_mn

The weight takes half the bytes of bf16, and the tensor cores run integers of 8
bits at twice the rate.  A row with a NaN or an infinity comes out as NaN.

Native path: ``_int8`` kernels.  Eager path (CPU tensors, or
``PD_KERNELS=eager``): the same integers in PyTorch.
"""
from __future__ import annotations

import os

import torch
import torch.nn.functional as F

from primus_dlrm_b200.ops import _ext
from primus_dlrm_b200.ops.saved8 import no_tangent

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_ACT = {None: 0, "": 0, "gelu": 1, "relu": 2}
MAX_FEATURES = 131072            # 128 * 127 * K stays below 2^31


def _native(t: torch.Tensor) -> bool:
    return t.is_cuda and os.environ.get("PD_KERNELS") != "eager"


def _quantize_ref(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True) if x.shape[-1] else x.new_zeros(*x.shape[:-1], 1)
    s = (amax * (1 / 127)).clamp(min=2.0 ** -126)
    s = torch.where(amax.isfinite(), s, torch.nan)
    codes = torch.round(torch.nan_to_num(x * (1 / s))).clamp(-127, 127).to(torch.int8)
    return codes, s.squeeze(-1)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Int8 codes of ``x`` ``[..., K]`` (bf16, fp16 or fp32) and the fp32 scale
    ``[...]`` of each row; ``codes * scale`` is within half a scale of ``x`` (and
    2^-15 of one, by the roundings of the scale and its reciprocal).  A row with
    a NaN or an infinity has codes of 0 and a scale of NaN.  Not differentiable:
    the results carry no graph."""
    if x.dim() == 0 or x.dtype not in _TYPES:
        raise ValueError(f"quantize_rows: a bf16, fp16 or fp32 tensor with a last dim is expected, not {x.dtype} of "
                         f"{x.dim()} dims")
    no_tangent("quantize_rows", x)
    x = x.detach()
    if not _native(x):
        return _quantize_ref(x)
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    x3 = x if x.dim() == 3 else x.reshape(x.shape[:-1].numel(), 1, x.shape[-1])
    codes, scale = _ext.int8().quantize_rows(x3)
    return codes.view(x.shape), scale.view(x.shape[:-1])


class Int8Weight:
    """A weight ``[N, K]`` (or ``[L, N, K]``: one for each of L token positions)
    as codes and channel scales.  Made by :meth:`from_float` or
    :meth:`from_tensors`."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, in_features: int, grouped: bool):
        # [L, N, K up to a multiple of 16, zeros behind K], [L, N]
        self._codes, self._scale, self.in_features, self.grouped = codes, scale, in_features, grouped

    @classmethod
    def from_tensors(cls, codes: torch.Tensor, scale: torch.Tensor) -> "Int8Weight":
        """From int8 codes ``[N, K]`` or ``[L, N, K]`` and fp32 scales ``[N]`` or ``[L, N]`` (not copied where codes are
        contiguous with K a multiple of 16)."""
        if codes.dtype != torch.int8 or codes.dim() not in (2, 3):
            raise ValueError("codes must be int8 [N, K] or [L, N, K]")
        if scale.dtype != torch.float32 or scale.shape != codes.shape[:-1] or scale.device != codes.device:
            raise ValueError("scale must be fp32 with one value for each row of codes, on their device")
        no_tangent("Int8Weight", scale)
        K = codes.shape[-1]
        if min(codes.shape) < 1 or K > MAX_FEATURES:
            raise ValueError(f"a weight of {tuple(codes.shape)}: 1 to {MAX_FEATURES} input features, and at least one "
                             "output feature, are expected")
        grouped = codes.dim() == 3
        codes, scale = (t if grouped else t.unsqueeze(0) for t in (codes.detach(), scale.detach().contiguous()))
        if K % 16 or not codes.is_contiguous() or codes.data_ptr() % 16:
            padded = codes.new_zeros(*codes.shape[:2], -(-K // 16) * 16)
            padded[..., :K] = codes
            codes = padded
        return cls(codes, scale, K, grouped)

    @classmethod
    def from_float(cls, weight: torch.Tensor) -> "Int8Weight":
        """From a bf16, fp16 or fp32 weight ``[N, K]`` or ``[L, N, K]``."""
        return cls.from_tensors(*quantize_rows(weight))

    @property
    def out_features(self) -> int:
        return self._codes.shape[1]

    @property
    def device(self) -> torch.device:
        return self._codes.device

    @property
    def codes(self) -> torch.Tensor:
        c = self._codes[..., :self.in_features]
        return c if self.grouped else c[0]

    @property
    def scale(self) -> torch.Tensor:
        return self._scale if self.grouped else self._scale[0]

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weight that the codes stand for."""
        return (self.codes.float() * self.scale[..., None]).to(dtype)


class _NoGradient(torch.autograd.Function):
    """An output of the integer product: a gradient asked of it raises."""

    @staticmethod
    def forward(ctx, y, *inputs):
        return y

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError("int8_linear has no gradient: call it under no_grad, or with detached inputs")


def _linear_ref(x, weight, bias, act, residual):
    a, s = _quantize_ref(x)
    w = weight.codes
    # products of integers below 2^53: exact in 64 bits
    acc = torch.einsum("...lk,lnk->...ln", a.double(), w.double()) if weight.grouped else a.double() @ w.double().t()
    y = acc.float() * (s[..., None] * weight.scale)
    if bias is not None:
        y = y + bias.float()
    y = F.gelu(y.clamp(min=-1e30)) if act == "gelu" else F.relu(y) if act == "relu" else y
    return (y + residual.float() if residual is not None else y).to(x.dtype)


def int8_linear(x: torch.Tensor, weight: Int8Weight, bias: torch.Tensor | None = None, act: str | None = None,
                residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x W^T + bias) + residual`` by 8-bit integers.

    ``x`` ``[..., K]`` is bf16, fp16 or fp32 with any strides (``[..., L, K]``
    where the weight has a matrix for each of L positions), ``bias`` ``[N]``,
    ``act`` None, ``"gelu"`` or ``"relu"``; ``residual`` has the result's shape
    ``[..., N]`` and ``x``'s type, which is the result's too.  A gradient asked
    of the result raises in the backward pass, a forward-mode tangent of an
    input at once.
    """
    code = _ACT.get(act)
    if code is None:
        raise ValueError(f"int8_linear: act {act!r}: expected None, 'gelu' or 'relu'")
    if x.is_cuda:
        y = _ext.int8().linear(x, weight._codes, weight._scale, weight.in_features, weight.grouped, bias, code, residual)
        if y is not None:                                    # None: PD_KERNELS=eager
            return y
    if x.dtype not in _TYPES:
        raise ValueError(f"int8_linear: {x.dtype}: expected bf16, fp16 or fp32")
    L = weight._codes.shape[0]
    if x.dim() < 1 + weight.grouped or x.shape[-1] != weight.in_features or (weight.grouped and x.shape[-2] != L):
        raise ValueError(f"int8_linear: x {tuple(x.shape)} does not fit a weight {tuple(weight.codes.shape)}")
    shape = (*x.shape[:-1], weight.out_features)
    if bias is not None and bias.shape != shape[-1:]:
        raise ValueError("int8_linear: bias must be [N]")
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype):
        raise ValueError("int8_linear: residual must have the result's shape and x's type")
    no_tangent("int8_linear", x, bias, residual)
    with torch.no_grad(), torch.autocast(x.device.type, enabled=False):
        y = _linear_ref(x, weight, bias, act, residual)
    inputs = [t for t in (x, bias, residual) if t is not None and t.requires_grad] if torch.is_grad_enabled() else []
    return _NoGradient.apply(y, *inputs) if inputs else y


def _err_word(device) -> torch.Tensor:
    device = torch.device(device)
    return _ext.int8().error_word(torch.cuda.current_device() if device.index is None else device.index)


def int8_error_code(device) -> int:
    """Error word of the integer products on ``device``, behind what the current
    stream holds (0 = ok, 2 = a bounded wait ran out, 4 = a block's shared
    memory was not aligned)."""
    return int(_err_word(device).item())


def check_errors(device) -> None:
    """Raises (and clears the word) if a product of integers on ``device`` gave
    up: results behind it are not to be used.  Waits for the current stream."""
    if torch.device(device).type != "cuda" or os.environ.get("PD_KERNELS") == "eager":
        return
    code = int8_error_code(device)
    if code:
        _err_word(device).zero_()
        raise RuntimeError({2: "int8_linear: a bounded wait in a kernel ran out",
                            4: "int8_linear: a kernel's shared memory is not aligned"}.get(
                                code, f"int8_linear: error {code}"))
