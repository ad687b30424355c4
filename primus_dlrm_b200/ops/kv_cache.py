"""Paged key/value cache in 8 bits, and attention over it.

A cache is a pool of pages of ``page_size`` tokens.  A page holds, for each
key/value head, ``page_size x d`` codes of e4m3 for keys and as many for
values, with one power-of-two scale each (``value = code * scale``): half the
memory and traffic of bf16.  A sequence's tokens lie in the pages that its row
of a page table names, in order; sequences may share pages (candidates that
follow one user's history), as long as nothing is appended to a shared page.

* :meth:`PagedKVCache.append` -- new tokens' keys and values, the keys normed
  and rotated on the way if asked;
* :meth:`PagedKVCache.read` -- tokens back as bf16 values;
* :func:`paged_attention` -- attention of each sequence's last tokens over
  its pages.

Native path: ``_kv`` kernels.  Eager path (CPU tensors, or
``PD_KERNELS=eager``): the same semantics in plain PyTorch.
"""
from __future__ import annotations

import math
import os

import torch

from primus_dlrm_b200.ops import _ext
from primus_dlrm_b200.ops.rotary import rotate_ref

_E4M3 = torch.float8_e4m3fn
_MIN_EXP = -100              # the smallest scale is 2^-100
PAGE_SIZES = (16, 32, 64)
HEAD_DIMS = (32, 64, 128)


def page_scale(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two (2^-100 at least) with ``amax / scale <= 448``."""
    f, e = torch.frexp(amax.float())
    e = torch.where(f > 0.875, e - 8, e - 9)
    return torch.ldexp(torch.ones_like(f), torch.where(amax > 0, e, _MIN_EXP).clamp(min=_MIN_EXP))


def _encode(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp32 values -> codes; non-finite values become NaN."""
    return torch.where(x.isfinite(), x / scale, torch.nan).clamp(-448, 448).to(_E4M3)


class PagedKVCache:
    """A pool of ``n_pages`` pages for ``n_kv_heads`` heads of ``head_dim``.

    ``k`` / ``v``: float8_e4m3fn ``[n_pages, n_kv_heads, page_size, head_dim]``;
    ``k_scale`` / ``v_scale``: fp32 ``[n_pages, n_kv_heads]``.  Which pages are
    in use is the caller's business.  ``page_size`` 16, 32 or 64, ``head_dim``
    32, 64 or 128.  Scales are finite and not negative.
    """

    def __init__(self, n_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64, device=None):
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        k = torch.zeros(shape, dtype=torch.uint8, device=device).view(_E4M3)
        scale = torch.full(shape[:2], 2.0 ** _MIN_EXP, device=device)
        self._set(k, torch.zeros_like(k.view(torch.uint8)).view(_E4M3), scale, scale.clone())

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor) -> "PagedKVCache":
        """A cache over existing codes and scales (not copied)."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        return self

    def _set(self, k, v, k_scale, v_scale):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != _E4M3 or v.dtype != _E4M3:
            raise ValueError("codes must be float8_e4m3fn [pages, heads, page_size, head_dim], keys and values alike")
        if k_scale.shape != k.shape[:2] or v_scale.shape != k.shape[:2]:
            raise ValueError("scales must be [pages, heads]")
        if k.shape[2] not in PAGE_SIZES:
            raise ValueError(f"page_size {k.shape[2]}: expected one of {PAGE_SIZES}")
        if k.shape[3] not in HEAD_DIMS:
            raise ValueError(f"head_dim {k.shape[3]}: expected one of {HEAD_DIMS}")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("codes and scales must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.err = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._parts = (k, v, k_scale, v_scale, self.err)
        self._cuda = k.is_cuda

    # ------------------------------------------------------------------
    @property
    def n_pages(self) -> int:
        return self.k.shape[0]

    @property
    def n_kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    @property
    def device(self) -> torch.device:
        return self.k.device

    def pages_for(self, tokens: int) -> int:
        """Pages that hold ``tokens`` tokens."""
        return -(-tokens // self.page_size)

    def check_errors(self) -> None:
        """Raises if a kernel met a page id outside the pool, a position outside
        the page table or the angle table, or an impossible length (such tokens
        are skipped on append, zeros on read and masked in attention; a token
        outside the angle table alone is kept with a key of zeros)."""
        e = int(self.err.item())
        if e:
            with torch.inference_mode():                # open to caches made in either mode
                self.err.zero_()
            raise RuntimeError({1: "paged cache: a page id, or a position, is out of range",
                                2: "paged cache: a bounded wait in a kernel ran out",
                                4: "paged cache: a kernel's shared memory is not aligned"}.get(
                                    e, "paged cache: a sequence's length does not fit its tokens or its page table"))

    def _native(self) -> bool:
        return self._cuda and os.environ.get("PD_KERNELS") != "eager"

    # ------------------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
               cu_new: torch.Tensor | None = None, max_new: int | None = None, *,
               k_weight: torch.Tensor | None = None, norm_eps: float | None = None,
               rope: torch.Tensor | None = None, interleaved: bool = False) -> None:
        """Writes new tokens behind the ``kv_lens[b]`` tokens that sequence ``b`` holds.

        ``k`` / ``v`` (bf16, fp16 or fp32, any strides over tokens and heads):
        ``[B, n, H, d]``, or ``[tokens, H, d]`` with ``cu_new`` int32 ``[B + 1]``,
        the offsets of each sequence's tokens; ``max_new`` is then the most of
        one sequence (by default all of them; a longer sequence is skipped and
        reported by :meth:`check_errors`).  ``page_table`` int32
        ``[B, pages]``, ``kv_lens`` int32 ``[B]`` (not changed).  No two
        sequences may write into one page.

        ``norm_eps``: the keys are normed per head (times ``k_weight``) first.
        ``rope``: an angle table of ``ops.rotary.rope_table`` with the head
        dim's width; the keys are then turned by their positions
        ``kv_lens[b] + i``.  Both in 32 bits.

        A page's scale is the smallest power of two that brings its largest
        finite magnitude to 448 or less; it never falls while the page fills,
        and where it grows the page's earlier tokens are rounded again.
        Non-finite values are stored as NaN and do not enter the scale.  No
        gradient passes through the cache: what it holds has none.
        """
        if self._native():
            _ext.kv().append(*self._parts, k, v, page_table, kv_lens, cu_new, max_new, k_weight, norm_eps, rope,
                             interleaved)
            return
        if k_weight is not None and norm_eps is None:
            raise ValueError("k_weight needs norm_eps")
        B = page_table.shape[0]
        if cu_new is None:
            if k.dim() != 4 or k.shape[0] != B:
                raise ValueError("k and v must be [sequences, tokens, heads, d]")
            parts = [(k[b], v[b]) for b in range(B)]
        else:
            o = cu_new.tolist()
            parts = [(k[a:e], v[a:e]) for a, e in zip(o, o[1:])]
        P = self.page_size
        for b, (kb, vb) in enumerate(parts):
            n, start = kb.shape[0], int(kv_lens[b])
            if n == 0:
                continue
            if start < 0 or start + n > page_table.shape[1] * P:
                raise ValueError(f"sequence {b}: {start} + {n} tokens do not fit its page table")
            kb, vb = kb.detach().float(), vb.detach().float()
            if norm_eps is not None:
                kb = kb * torch.rsqrt(kb.pow(2).mean(-1, keepdim=True) + norm_eps)
                kb = kb if k_weight is None else kb * k_weight.detach().float()
            if rope is not None:
                if start + n > rope.shape[0]:
                    raise IndexError(f"a position lies outside the angle table of {rope.shape[0]} rows")
                kb = rotate_ref(kb, rope[start:start + n], interleaved)
            for j in range(start // P, (start + n - 1) // P + 1):
                lo, hi = max(start, j * P), min(start + n, (j + 1) * P)
                page = self._page(page_table, b, j)
                for x, code, scale in ((kb, self.k, self.k_scale), (vb, self.v, self.v_scale)):
                    y = x[lo - start:hi - start].transpose(0, 1)                       # [H, rows, d]
                    s = page_scale(torch.where(y.isfinite(), y.abs(), 0.0).amax((1, 2)))
                    r = lo - j * P
                    if r > 0:
                        s = torch.maximum(s, scale[page])
                        held = code[page, :, :r].float() * scale[page][:, None, None]
                        code[page, :, :r] = _encode(held, s[:, None, None])
                    code[page, :, r:hi - j * P] = _encode(y, s[:, None, None])
                    scale[page] = s

    def _page(self, page_table, b: int, j: int) -> int:
        p = int(page_table[b, j])
        if not 0 <= p < self.n_pages:
            raise IndexError(f"sequence {b}: page id {p} is out of range")
        return p

    def read(self, page_table: torch.Tensor, kv_lens: torch.Tensor, first: torch.Tensor | None = None,
             n: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Tokens ``first[b] .. first[b] + n - 1`` of each sequence as the values
        that their codes stand for: two bf16 ``[B, n, H, d]``, zeros behind
        ``kv_lens[b]``.  By default every token that the page table has room for."""
        if self._native():
            return tuple(_ext.kv().read(*self._parts, page_table, kv_lens, first, n))
        if n is None:
            n = page_table.shape[1] * self.page_size
        B, P = page_table.shape[0], self.page_size
        out = [torch.zeros(B, n, self.n_kv_heads, self.head_dim, dtype=torch.bfloat16, device=self.device)
               for _ in range(2)]
        for b in range(B):
            f, e = int(first[b]) if first is not None else 0, int(kv_lens[b])
            for pos in range(max(f, 0), min(f + n, e)):
                page = self._page(page_table, b, pos // P)
                for o, code, scale in ((out[0], self.k, self.k_scale), (out[1], self.v, self.v_scale)):
                    o[b, pos - f] = (code[page, :, pos % P].float() * scale[page][:, None]).to(torch.bfloat16)
        return out[0], out[1]

    @torch.no_grad()
    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Pages ``dst`` become copies of pages ``src`` (integers ``[n]`` each, ``dst``
        all different): how a sequence gets a page of its own before it appends
        behind a shared one.  Every source is read before the first page is
        written.  A pair with an id outside the pool is skipped and reported by
        :meth:`check_errors` (IndexError on the eager path)."""
        src, dst = torch.broadcast_tensors(torch.as_tensor(src), torch.as_tensor(dst))
        if src.numel() and any(t.dtype == torch.bool or t.is_floating_point() for t in (src, dst)):
            raise TypeError("page ids must be integers")
        src, dst = (t.to(self.device, torch.int64).reshape(-1) for t in (src, dst))
        if self._native():
            _ext.kv().copy_pages(*self._parts, src.contiguous(), dst.contiguous())
            return
        for t in (src, dst):
            if t.numel() and not 0 <= int(t.min()) <= int(t.max()) < self.n_pages:
                raise IndexError(f"a page id lies outside the pool of {self.n_pages}")
        for t in (self.k.view(torch.uint8), self.v.view(torch.uint8), self.k_scale, self.v_scale):
            t[dst] = t[src]


def paged_attention_ref(q, cache: PagedKVCache, page_table, kv_lens, cu_q=None, scale: float | None = None,
                        causal: bool = True, dtype=torch.float32):
    """Plain attention over a cache: (o, lse) in ``dtype``, one sequence and head at a time."""
    d = cache.head_dim
    scale = d ** -0.5 if scale is None else scale
    B, P = page_table.shape[0], cache.page_size
    flat = q.reshape(-1, *q.shape[-2:])
    Hq = flat.shape[1]
    off = cu_q.tolist() if cu_q is not None else [b * q.shape[1] for b in range(B + 1)]
    o = torch.zeros(flat.shape, dtype=dtype, device=q.device)
    lse = torch.full(flat.shape[:2], -math.inf, dtype=dtype, device=q.device)
    for b in range(B):
        n, length = off[b + 1] - off[b], int(kv_lens[b])
        if n <= 0 or length <= 0:
            continue
        ids = [cache._page(page_table, b, j) for j in range(-(-length // P))]
        kv = []
        for code, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            x = code.view(torch.uint8)[ids].view(_E4M3).to(dtype) * s[ids].to(dtype)[..., None, None]
            kv.append(x.transpose(0, 1).flatten(1, 2)[:, :length].repeat_interleave(Hq // cache.n_kv_heads, 0))
        qb = flat[off[b]:off[b + 1]].to(dtype).transpose(0, 1)
        w = qb @ kv[0].transpose(1, 2) * scale
        if causal:
            last = length - n + torch.arange(n, device=q.device)
            w = w.masked_fill(torch.arange(length, device=q.device) > last[:, None], -math.inf)
        z = torch.logsumexp(w, -1)
        p = torch.where(z[..., None] == -math.inf, 0.0, torch.exp(w - z[..., None]))
        o[off[b]:off[b + 1]] = (p @ kv[1]).transpose(0, 1)
        lse[off[b]:off[b + 1]] = z.transpose(0, 1)
    return o.reshape(q.shape), lse.reshape(q.shape[:-1])


class _NoGradient(torch.autograd.Function):
    """Results of a query that requires a gradient: the backward pass says that there is none."""

    @staticmethod
    def forward(ctx, q, *out):
        return tuple(x.view_as(x) for x in out)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("paged_attention has no gradient: call it under no_grad, or with a detached query")


def paged_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, kv_lens: torch.Tensor,
                    cu_q: torch.Tensor | None = None, max_q: int | None = None, *, max_len: int | None = None,
                    scale: float | None = None, causal: bool = True, return_lse: bool = False):
    """Attention of each sequence's last tokens over the cache (no gradient: a
    backward pass through it raises, as do forward-mode tangents).

    ``q`` (bf16 or fp16, any strides over tokens and heads): ``[B, n, Hq, d]``,
    or ``[tokens, Hq, d]`` with ``cu_q`` int32 ``[B + 1]``; ``max_q`` is then the
    most queries of one sequence (by default all of them; a longer sequence is
    skipped and reported by ``cache.check_errors``; its rows, and those of ``q``
    that no sequence covers, give zeros and ``-inf``).  ``Hq`` is a
    multiple of the cache's heads: neighbours share one.  ``kv_lens`` int32
    ``[B]`` counts the tokens in the cache, the queries' own among them, so a
    sequence's ``n`` queries are its last ``n`` tokens: query ``i`` sees the
    keys ``j <= kv_lens[b] - n + i``, or with ``causal=False`` all of them.
    ``max_len`` is an upper bound of ``kv_lens`` (by default the page table's
    room); it only decides how the work is split.  State it, and ``max_q``, where
    they are known: from the defaults a slower form may be chosen.  ``scale`` is ``d ** -0.5``
    unless given.

    Returns ``o`` like ``q`` (contiguous), or ``(o, lse)`` with the natural
    log-sum-exp of the scaled scores in fp32.  A query without keys gives
    zeros and ``-inf``.
    """
    if cache._native():
        out = _ext.kv().paged_attention(q, *cache._parts, page_table, kv_lens, cu_q, max_q, max_len, scale, causal,
                                        return_lse)
        return (out[0], out[1]) if return_lse else out[0]
    if torch.autograd.forward_ad.unpack_dual(q).tangent is not None:
        raise RuntimeError("paged_attention has no forward-mode derivative")
    o, lse = paged_attention_ref(q.detach(), cache, page_table, kv_lens, cu_q, scale, causal)
    o = o.to(q.dtype)
    if torch.is_grad_enabled() and q.requires_grad:
        o, lse = _NoGradient.apply(q, o, lse)
    return (o, lse) if return_lse else o
