"""OneTrans: one causal Transformer over behaviour-sequence (S) and
non-sequential (NS) tokens.

Architecture and parameter layout follow ``primus_dlrm/models/onetrans.py``
(so checkpoints interchange key-for-key):

* per-group ``SequentialTokenizer`` (Linear(G*E, D) -> GELU -> Linear(D, D)
  + learned positions) builds the S tokens (``onetrans.py:238-257``);
* ``AutoSplitTokenizer`` maps the concatenated NS features to ``n_ns`` tokens
  (``onetrans.py:260-276``);
* blocks use *mixed parameterisation*: S tokens share ``s_qkv`` / ``s_w1`` /
  ``s_w2``, each NS token has its own slice of ``ns_qkv_weight`` /
  ``ns_w1`` / ``ns_w2`` (``onetrans.py:85-204``);
* pyramid query pruning: layer ``l`` keeps the last ``schedule[l] + n_ns``
  queries and attends bottom-right causally (``onetrans.py:50-67``).

Execution (B200): the lookup writes every pool's ``[B, L, 3E]`` tokenizer
input in bf16 with one kernel; the S and NS projections write into one
``[B, T, 3D]`` QKV buffer (no concatenation); norm kernels fuse the
attention residual; heads + multi-task loss are one fused op.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from primus_dlrm_b200.config import Config
from primus_dlrm_b200.models.base import BaseModel
from primus_dlrm_b200.models.embedding import Embeddings
from primus_dlrm_b200.models.heads import fused_heads_loss
from primus_dlrm_b200.ops import dense, int8
from primus_dlrm_b200.ops.attention import (
    _native_ok as _fmha_native_ok, causal_attention_all_rows, pyramid_attention, pyramid_attention_qkv,
)
from primus_dlrm_b200.ops.embedding import SparseOptimizer
from primus_dlrm_b200.ops.int8 import Int8Weight, int8_linear
from primus_dlrm_b200.ops.kv_cache import PagedKVCache, paged_attention
from primus_dlrm_b200.ops.norm import RMSNorm, add_norm, make_norm, norm_with_tail
from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table


def pyramid_schedule(l_s: int, l_ns: int, n_layers: int) -> list[int]:
    """S-token query count per layer, shrinking linearly from ``l_s`` to
    ``l_ns`` (rounded, floored at ``l_ns``; one layer keeps ``l_ns``)."""
    if n_layers <= 1:
        return [l_ns]
    step = (l_s - l_ns) / (n_layers - 1)
    return [max(int(round(l_s - i * step)), l_ns) for i in range(n_layers)]


def _xavier_per_token(w: torch.Tensor) -> None:
    for i in range(w.shape[0]):
        nn.init.xavier_uniform_(w.data[i])


class MixedAttention(nn.Module):
    def __init__(self, d_model: int, n_heads: int, n_ns_tokens: int, dropout: float = 0.0,
                 attention_impl: str = "sdpa", rotary: bool = False, rope_theta: float = 10000.0,
                 save8: bool = False):
        super().__init__()
        if d_model % n_heads:
            raise ValueError("d_model must be divisible by n_heads")
        if attention_impl not in ("sdpa", "fav2", "fav4", "turbo", "native", "mask"):
            raise ValueError(f"Unknown attention_impl: {attention_impl!r}. "
                             f"Supported: 'sdpa', 'fav2', 'fav4', 'turbo', 'native'")
        self.d_model = d_model
        self.n_heads = n_heads
        self.d_head = d_model // n_heads
        self.n_ns = n_ns_tokens
        self.attention_impl = attention_impl
        self.s_qkv = nn.Linear(d_model, 3 * d_model, bias=False)
        self.ns_qkv_weight = nn.Parameter(torch.empty(n_ns_tokens, 3 * d_model, d_model))
        self.out_proj = nn.Linear(d_model, d_model, bias=False)
        self.attn_drop = dropout
        nn.init.xavier_uniform_(self.s_qkv.weight)
        nn.init.xavier_uniform_(self.out_proj.weight)
        _xavier_per_token(self.ns_qkv_weight)
        self.rotary, self.rope_theta, self.save8 = rotary, rope_theta, save8
        if rotary:
            self.q_norm, self.k_norm = RMSNorm(self.d_head), RMSNorm(self.d_head)
            self._rope: torch.Tensor | None = None

    def rope(self, tokens: int, device) -> torch.Tensor:
        """Angle table of at least ``tokens`` positions."""
        if self._rope is None or self._rope.shape[0] < tokens or self._rope.device != torch.device(device):
            with torch.inference_mode(False):                # a later training step saves it for its backward
                self._rope = rope_table(max(256, 1 << (tokens - 1).bit_length()), self.d_head, self.rope_theta, device)
        return self._rope

    def norm_rope(self, q: torch.Tensor, k: torch.Tensor | None, tokens: int) -> tuple[torch.Tensor, torch.Tensor | None]:
        """q (the last rows) and k of a ``tokens`` long sequence, normed per head and rotated."""
        table = self.rope(tokens, q.device)
        pos = None if k is not None else torch.arange(tokens - q.shape[1], tokens, device=q.device)
        return qk_norm_rope(q, k, self.q_norm.weight, self.k_norm.weight, table, pos, eps=self.q_norm.eps)

    def forward(self, x: torch.Tensor, n_s: int, q_len: int) -> torch.Tensor:
        """x [B, T, D] (normed) -> out-projected attention of the last q_len
        queries, [B, q_len, D].  On CUDA (no dropout, native impls) all T rows
        are computed and the result is a [B, q_len, D] view of [B, T, D]."""
        B, T, D = x.shape
        qkv = dense.mixed_linear(x, n_s, self.s_qkv.weight, self.ns_qkv_weight, save8=self.save8)  # [B, T, 3D]
        qkv = qkv.view(B, T, 3, self.n_heads, self.d_head)
        if self.rotary:
            q, k = self.norm_rope(qkv[:, T - q_len:, 0], qkv[:, :, 1], T)
            impl = "mask" if not x.is_cuda or self.attention_impl in ("sdpa", "mask") else "auto"
            drop = self.attn_drop if (self.training and self.attention_impl in ("sdpa", "fav2", "turbo")) else 0.0
            out = pyramid_attention(q, k, qkv[:, :, 2].contiguous(), impl=impl, dropout_p=drop)
            return dense.linear(self.out_proj, out.reshape(B, q_len, D))
        no_drop = not (self.training and self.attn_drop > 0 and self.attention_impl != "fav4")
        if x.is_cuda and self.attention_impl in ("fav4", "fav2", "turbo", "native") and no_drop \
                and _fmha_native_ok(qkv):
            o = pyramid_attention_qkv(qkv, q_len)
            return dense.linear(self.out_proj, o.reshape(B, q_len, D))
        if x.is_cuda and self.attention_impl in ("fav4", "fav2", "turbo", "native") and \
                not (self.training and self.attn_drop > 0 and self.attention_impl != "fav4"):
            o = causal_attention_all_rows(qkv, self.n_heads).reshape(B, T, D)
            return self.out_proj(o)[:, T - q_len:]
        q = qkv[:, T - q_len:, 0]
        k = qkv[:, :, 1]
        v = qkv[:, :, 2]
        impl = {"sdpa": "mask", "native": "native"}.get(self.attention_impl, "auto")
        if not x.is_cuda:
            impl = "mask"
        drop = self.attn_drop if (self.training and self.attention_impl in ("sdpa", "fav2", "turbo")) else 0.0
        out = pyramid_attention(q, k, v, impl=impl, dropout_p=drop)
        return self.out_proj(out.reshape(B, q_len, D))


class MixedFFN(nn.Module):
    def __init__(self, d_model: int, ffn_dim: int, n_ns_tokens: int, dropout: float = 0.0, save8: bool = False):
        super().__init__()
        self.n_ns, self.save8 = n_ns_tokens, save8
        self.d_model = d_model
        self.s_w1 = nn.Linear(d_model, ffn_dim, bias=False)
        self.s_w2 = nn.Linear(ffn_dim, d_model, bias=False)
        self.ns_w1 = nn.Parameter(torch.empty(n_ns_tokens, ffn_dim, d_model))
        self.ns_w2 = nn.Parameter(torch.empty(n_ns_tokens, d_model, ffn_dim))
        self.dropout = nn.Dropout(dropout)
        nn.init.xavier_uniform_(self.s_w1.weight)
        nn.init.xavier_uniform_(self.s_w2.weight)
        _xavier_per_token(self.ns_w1)
        _xavier_per_token(self.ns_w2)

    def forward(self, x: torch.Tensor, n_s: int) -> torch.Tensor:
        h = dense.mixed_linear(x, n_s, self.s_w1.weight, self.ns_w1, act="gelu", save8=self.save8)
        h = self.dropout(h)
        return dense.mixed_linear(h, n_s, self.s_w2.weight, self.ns_w2, save8=self.save8)


class OneTransBlock(nn.Module):
    """Pre-norm block: z = x_tail + Attn(N1(x)); out = z + FFN(N2(z))."""

    def __init__(self, d_model: int, n_heads: int, n_ns_tokens: int, ffn_mult: int = 4,
                 dropout: float = 0.0, attention_impl: str = "sdpa", norm: str = "rmsnorm", rotary: bool = False,
                 rope_theta: float = 10000.0, activation_bits: int = 16):
        super().__init__()
        if activation_bits not in (8, 16):
            raise ValueError(f"activation_bits {activation_bits}: expected 16 or 8")
        save8 = activation_bits == 8
        self.norm1 = make_norm(norm, d_model)
        self.attn = MixedAttention(d_model, n_heads, n_ns_tokens, dropout, attention_impl, rotary, rope_theta, save8)
        self.norm2 = make_norm(norm, d_model)
        self.ffn = MixedFFN(d_model, d_model * ffn_mult, n_ns_tokens, dropout, save8)

    def forward(self, x: torch.Tensor, q_len: int, n_s_tokens: int) -> torch.Tensor:
        kv_len = x.shape[1]
        n_ns = kv_len - n_s_tokens
        h, x_tail = norm_with_tail(self.norm1, x, q_len)
        a = self.attn(h, n_s=n_s_tokens, q_len=q_len)
        y, z = add_norm(a, x_tail, self.norm2.weight,
                        getattr(self.norm2, "bias", None), self.norm2.eps, self.norm2.kind)
        fused = dense.mixed_ffn(y, z, q_len - n_ns, self.ffn.s_w1.weight, self.ffn.s_w2.weight,
                                self.ffn.ns_w1, self.ffn.ns_w2, save8=self.ffn.save8) if (self.ffn.dropout.p == 0 or not self.training) else None
        if fused is not None:
            return fused
        f = self.ffn(y, n_s=q_len - n_ns)
        return z + f


class SequentialTokenizer(nn.Module):
    def __init__(self, raw_dim: int, d_model: int, max_len: int = 1024, use_pos_embed: bool = True):
        super().__init__()
        self.proj = nn.Sequential(nn.Linear(raw_dim, d_model), nn.GELU(), nn.Linear(d_model, d_model))
        self.pos_emb = nn.Embedding(max_len, d_model) if use_pos_embed else None

    def forward(self, raw: torch.Tensor) -> torch.Tensor:
        pos = self.pos_emb.weight[: raw.shape[1]] if self.pos_emb is not None else None
        return dense.mlp2(raw, self.proj[0], self.proj[2], addend=pos)


class AutoSplitTokenizer(nn.Module):
    def __init__(self, ns_input_dim: int, d_model: int, n_ns_tokens: int):
        super().__init__()
        out = d_model * n_ns_tokens
        self.proj = nn.Sequential(nn.Linear(ns_input_dim, out), nn.GELU(), nn.Linear(out, out))
        self.n_ns_tokens = n_ns_tokens
        self.d_model = d_model

    def forward(self, ns: torch.Tensor) -> torch.Tensor:
        return dense.mlp2(ns, self.proj[0], self.proj[2]).view(-1, self.n_ns_tokens, self.d_model)


class _UserPages:
    """One layer's 8-bit pages for scoring: a user's history, then the tokens of
    up to ``slots`` candidates behind it at a time."""

    def __init__(self, attn: MixedAttention, n_s: int, n_ns: int, slots: int, device):
        self.attn, self.n_s, self.n_ns = attn, n_s, n_ns
        P = 64
        full, tail = divmod(n_s, P)                          # the history's full pages, tokens in the one behind
        own = -(-(tail + n_ns) // P)                         # pages of a candidate
        shared = full + (tail > 0)
        self.cache = PagedKVCache(shared + slots * own, attn.n_heads, attn.d_head, P, device=device)
        first = torch.arange(shared, dtype=torch.int32, device=device)
        mine = shared + torch.arange(slots * own, dtype=torch.int32, device=device).view(slots, own)
        self.history_table = first[None]
        self.table = torch.cat([first[:full].expand(slots, -1), mine], dim=1)
        self.tail = (first[full:].long().expand(slots), mine[:, 0].long()) if tail else None
        self.norm = {}
        if attn.rotary:
            self.norm = dict(k_weight=attn.k_norm.weight, norm_eps=attn.k_norm.eps, rope=attn.rope(n_s + n_ns, device))

    def _attend(self, q, table, tokens: int):
        """The last rows' attention over ``tokens`` tokens of each sequence."""
        lens = torch.full((q.shape[0],), tokens, dtype=torch.int32, device=q.device)
        if self.attn.rotary:
            q, _ = self.attn.norm_rope(q, None, tokens)
        half = q.dtype if q.dtype in (torch.bfloat16, torch.float16) or not q.is_cuda else torch.bfloat16
        return paged_attention(q.to(half), self.cache, table, lens, max_len=tokens).to(q.dtype)

    def _append(self, k, v, table, held: int):
        lens = torch.full((k.shape[0],), held, dtype=torch.int32, device=k.device)
        self.cache.append(k, v, table, lens, **self.norm)

    def history(self, q, k, v):
        """Attention of the history's last queries; its keys and values stay in the cache."""
        self._append(k, v, self.history_table, 0)
        return self._attend(q, self.history_table, self.n_s)

    def candidates(self, q, k, v):
        """Attention of each candidate's tokens over the history and themselves."""
        table = self.table[:q.shape[0]]
        if self.tail is not None:                            # a copy of the partly filled page for each candidate
            self.cache.copy_pages(self.tail[0][:q.shape[0]], self.tail[1][:q.shape[0]])
        self._append(k, v, table, self.n_s)
        return self._attend(q, table, self.n_s + self.n_ns)


class OneTransModel(BaseModel):
    def __init__(self, config: Config, device: torch.device | None = None, meta_device: bool = False):
        super().__init__()
        self.config = config
        mc, fc, ot = config.model, config.feature, config.model.transformer
        device = torch.device("cpu") if device is None else torch.device(device)
        emb_device = torch.device("meta") if meta_device else device
        self.tasks = list(config.task_names)
        E = mc.embedding_dim
        tc = config.train
        opt = SparseOptimizer(kind=tc.embedding_optimizer, lr=tc.embedding_lr, eps=tc.embedding_eps,
                              weight_decay=tc.weight_decay)
        self.emb = Embeddings(mc.resolved_embedding_tables(), device=emb_device,
                              embedding_init=mc.embedding_init,
                              scalar_feature_names=set(fc.scalar_feature_names), optimizer=opt)
        self.seq_tokenizers = nn.ModuleDict({
            g: SequentialTokenizer(sum(self.emb.feature_dim(f) for f in feats), ot.d_model, max_len=2048,
                                   use_pos_embed=ot.pos_embed)
            for g, feats in fc.sequence_groups.items()
        }).to(device)
        self.dense_projs = nn.ModuleDict()
        ns_raw = sum(self.emb.feature_dim(f) for f in fc.scalar_feature_names)
        for df in fc.dense_features:
            if df.project:
                act = nn.ReLU(inplace=True) if df.activation == "relu" else nn.GELU()
                self.dense_projs[df.name] = nn.Sequential(nn.Linear(df.dim, E, device=device), act)
                ns_raw += E
            else:
                ns_raw += df.dim
        self.ns_raw_dim = ns_raw
        self.ns_tokenizer = AutoSplitTokenizer(ns_raw, ot.d_model, ot.n_ns_tokens).to(device)
        self.blocks = nn.ModuleList([
            OneTransBlock(ot.d_model, ot.n_heads, ot.n_ns_tokens, ot.ffn_mult, ot.dropout,
                          attention_impl=ot.attention_impl, norm=ot.norm, rotary=ot.rotary, rope_theta=ot.rope_theta,
                          activation_bits=ot.activation_bits)
            for _ in range(ot.n_layers)
        ]).to(device)
        self.final_norm = make_norm(ot.norm, ot.d_model).to(device)
        self.head_proj = nn.Sequential(nn.Linear(ot.n_ns_tokens * ot.d_model, ot.d_model, device=device),
                                       nn.GELU(), nn.Dropout(ot.dropout))
        self.heads = nn.ModuleDict({t: nn.Linear(ot.d_model, 1, device=device) for t in self.tasks})
        self._item_scalar_names = [s.name for s in fc.item_scalar_features]
        self.contrastive_user_proj = nn.Linear(ot.d_model, ot.d_model, device=device)
        self.contrastive_item_proj = nn.Sequential(
            nn.Linear(sum(self.emb.feature_dim(f) for f in self._item_scalar_names) or 1, ot.d_model,
                      device=device), nn.ReLU(inplace=True))

    # ------------------------------------------------------------------
    def get_num_flops_per_sample(self) -> float:
        """Analytic fwd+bwd FLOPs per sample (6x per matmul MAC, 12x attention,
        no causal discount); same accounting as ``onetrans.py:392-474`` with
        per-group history lengths."""
        cfg = self.config
        ot, fc = cfg.model.transformer, cfg.feature
        D, H, n_ns = ot.d_model, ot.n_heads, ot.n_ns_tokens
        dh, F_ = D // H, D * ot.ffn_mult
        L_S = cfg.sequence_length_total()
        sched = pyramid_schedule(L_S, n_ns, ot.n_layers) if ot.use_pyramid else [L_S] * ot.n_layers
        fl = 0
        for g, feats in fc.sequence_groups.items():
            raw = sum(self.emb.feature_dim(f) for f in feats)
            fl += 6 * cfg.data.group_length(g) * (raw * D + D * D)
        for df in fc.dense_features:
            if df.project:
                fl += 6 * df.dim * cfg.model.embedding_dim
        no = n_ns * D
        fl += 6 * (self.ns_raw_dim * no + no * no)
        kv = L_S + n_ns
        for l in range(ot.n_layers):
            q = sched[l] + n_ns
            fl += 6 * (kv - n_ns) * D * 3 * D + 6 * n_ns * 3 * D * D
            fl += 12 * H * dh * q * kv
            fl += 6 * q * D * D
            fl += 6 * (q - n_ns) * D * F_ * 2 + 6 * n_ns * D * F_ * 2
            kv = q
        fl += 6 * n_ns * D * D + 6 * len(self.tasks) * D
        if cfg.train.contrastive_weight > 0:
            fl += 6 * D * D + 6 * len(self._item_scalar_names) * cfg.model.embedding_dim * D
            fl += 6 * D * (cfg.train.batch_size // (cfg.distributed.num_nodes * cfg.distributed.gpus_per_node))
        return float(fl)

    # ------------------------------------------------------------------
    def _compute_dtype(self, batch) -> torch.dtype:
        return torch.bfloat16 if (torch.is_autocast_enabled("cuda") or torch.is_autocast_enabled("cpu")) \
            else torch.float32

    def _lookup(self, batch: dict[str, torch.Tensor]):
        """One fused lookup: every pool's [B, L, G*E] input + the [B, n_scalar*E] NS block."""
        f2k = self.config.feature_to_batch_key()
        fc = self.config.feature
        feats = {}
        for f in fc.all_ec_feature_names():
            k = f2k.get(f, f)
            if k in batch:
                feats[f] = batch[k]
        groups = [list(v) for v in fc.sequence_groups.values()] + [list(fc.scalar_feature_names)]
        outs = self.emb.lookup_groups(feats, groups, dtype=self._compute_dtype(batch))
        return outs[:-1], outs[-1]

    def _backbone(self, batch: dict[str, torch.Tensor]):
        ot = self.config.model.transformer
        pools, scal = self._lookup(batch)
        s_parts = [tok(raw) for tok, raw in zip(self.seq_tokenizers.values(), pools)]
        parts = [scal]
        for df in self.config.feature.dense_features:
            x = batch[df.name]
            parts.append(self._dense_proj(df, x, scal.dtype) if df.name in self.dense_projs else x.to(scal.dtype))
        ns_raw = torch.cat([p.to(scal.dtype) for p in parts], dim=-1)
        ns_tokens = self.ns_tokenizer(ns_raw)
        # one concatenation of every S pool's tokens and the NS tokens
        x = torch.cat(s_parts + [ns_tokens.to(s_parts[0].dtype)], dim=1)
        B = x.shape[0]
        L_NS = ot.n_ns_tokens
        L_S = x.shape[1] - L_NS
        sched = pyramid_schedule(L_S, L_NS, ot.n_layers) if ot.use_pyramid else [L_S] * ot.n_layers
        for l, block in enumerate(self.blocks):
            q_len = sched[l] + L_NS
            x = block(x, q_len=q_len, n_s_tokens=x.shape[1] - L_NS)
        x = self.final_norm(x)
        s_repr = x[:, : x.shape[1] - L_NS].float().mean(dim=1)
        hp = self.head_proj
        h = hp[2](dense.linear(hp[0], x[:, -L_NS:].reshape(B, -1), act="gelu"))
        return h, s_repr, scal

    def _dense_proj(self, df, x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        """Linear + activation of a projected dense feature (GEMM epilogue on CUDA)."""
        seq = self.dense_projs[df.name]
        act = "relu" if isinstance(seq[1], nn.ReLU) else "gelu"
        return dense.linear(seq[0], x.to(dtype), act=act)

    def forward(self, batch: dict[str, torch.Tensor]) -> dict[str, torch.Tensor]:
        h, _, _ = self._backbone(batch)
        return {t: head(h).squeeze(-1) for t, head in self.heads.items()}

    def forward_loss(self, batch: dict[str, torch.Tensor], loss_weights: dict[str, float],
                     regression_tasks: list[str]):
        """(total, {task: loss}, {task: logits}) with heads + loss fused."""
        h, _, _ = self._backbone(batch)
        return fused_heads_loss(self.heads, h, batch, loss_weights, regression_tasks)

    # ------------------------------------------------------------------
    @torch.no_grad()
    def int8_weights(self) -> list[dict[str, Int8Weight]]:
        """The blocks' projection weights as 8-bit integers, for :meth:`score_candidates`; later training steps do not
        reach them."""
        return [{"s_qkv": Int8Weight.from_float(b.attn.s_qkv.weight), "ns_qkv": Int8Weight.from_float(b.attn.ns_qkv_weight),
                 "out": Int8Weight.from_float(b.attn.out_proj.weight), "s_w1": Int8Weight.from_float(b.ffn.s_w1.weight),
                 "s_w2": Int8Weight.from_float(b.ffn.s_w2.weight), "ns_w1": Int8Weight.from_float(b.ffn.ns_w1),
                 "ns_w2": Int8Weight.from_float(b.ffn.ns_w2)} for b in self.blocks]

    @torch.no_grad()
    def score_candidates(self, user_batch: dict[str, torch.Tensor], candidate_batch: dict[str, torch.Tensor],
                         task: str, batch_size: int = 1024, kv_cache: str | None = None,
                         weights: list[dict[str, Int8Weight]] | None = None) -> torch.Tensor:
        """Scores [C] of one user against C candidates with an S-side K/V cache.

        S tokens sit before the NS tokens and attention is causal, so the S
        stream (hidden states, and the keys / values of every layer) depends
        on the user's history only: it is computed once, for a batch of one,
        following the pyramid. Each candidate then runs only its NS tokens,
        attending to the cached S keys / values plus its own NS keys -- the
        same function as ``forward`` on (user history, candidate), at the cost
        of n_ns tokens per candidate instead of L_S + n_ns
        (``primus_dlrm/evaluation/metrics.py:200-279`` recomputes everything).

        ``kv_cache="fp8"`` keeps the keys and values in pages of 8 bits
        (``ops.kv_cache``): every candidate's page table names the user's full
        pages, and only the last, partly filled one is copied, instead of
        expanding the cache to each candidate.  The head dim is then 32, 64 or
        128, and scores carry the rounding of 8-bit keys and values; on a GPU the
        queries and outputs of a 32-bit model are rounded to bf16 there.

        ``weights`` (:meth:`int8_weights`, laid out once for many users) runs the
        blocks' projections as products of 8-bit integers (``ops.int8``); scores
        carry the rounding of 8-bit weights and activations.
        """
        if kv_cache not in (None, "fp8"):
            raise ValueError(f"kv_cache {kv_cache!r}: expected None or 'fp8'")
        if weights is not None and len(weights) != len(self.blocks):
            raise ValueError(f"weights of {len(weights)} blocks for a model of {len(self.blocks)}")
        ot = self.config.model.transformer
        n_ns, H = ot.n_ns_tokens, ot.n_heads
        D = ot.d_model
        dh = D // H
        C = next(iter(candidate_batch.values())).shape[0]
        # ---- user side: S tokens through the pyramid, caching per-layer K / V ----
        f2k = self.config.feature_to_batch_key()
        fc = self.config.feature
        seq = {f: user_batch[f2k.get(f, f)] for feats in fc.sequence_groups.values() for f in feats}
        pools = self.emb.lookup_groups(seq, [list(v) for v in fc.sequence_groups.values()],
                                       dtype=self._compute_dtype(user_batch))
        xs = torch.cat([tok(raw) for tok, raw in zip(self.seq_tokenizers.values(), pools)], dim=1)  # [1, L_S, D]
        L_S = xs.shape[1]
        sched = pyramid_schedule(L_S, n_ns, ot.n_layers) if ot.use_pyramid else [L_S] * ot.n_layers
        cache = []
        for l, blk in enumerate(self.blocks):
            at = blk.attn
            h = blk.norm1(xs)
            w8 = weights[l] if weights else None
            qkv = int8_linear(h, w8["s_qkv"]) if w8 else h @ at.s_qkv.weight.t().to(h.dtype)
            qkv = qkv.view(1, -1, 3, H, dh)
            q_s = sched[l]                                   # S queries kept by this layer
            k_s, v_s = qkv[:, :, 1], qkv[:, :, 2]            # [1, n_s, H, dh]
            n_s = xs.shape[1]
            q = qkv[:, n_s - q_s:, 0]
            if kv_cache:
                cache.append(_UserPages(at, n_s, n_ns, min(C, batch_size), xs.device))
                o = cache[-1].history(q, k_s, v_s).reshape(1, q_s, D)
            else:
                if at.rotary:
                    q, k_s = at.norm_rope(q, k_s, n_s)
                cache.append((k_s, v_s))
                o = pyramid_attention(q, k_s, v_s, impl="mask").reshape(1, q_s, D)
            tail = xs[:, n_s - q_s:]
            if w8:
                z = int8_linear(o, w8["out"], residual=tail.to(o.dtype))
                f = int8_linear(blk.norm2(z), w8["s_w1"], act="gelu")
                xs = int8_linear(f, w8["s_w2"], residual=z.to(f.dtype))
                continue
            z = at.out_proj(o) + tail
            y = blk.norm2(z)
            xs = z + blk.ffn.s_w2(F.gelu(blk.ffn.s_w1(y)))
        # ---- candidate side: NS tokens only ----
        scores = []
        for c0 in range(0, C, batch_size):
            c1 = min(C, c0 + batch_size)
            cb = {k: v[c0:c1] for k, v in candidate_batch.items()}
            nb = c1 - c0
            for k, v in user_batch.items():
                if k not in cb:
                    cb[k] = v.expand(nb, *v.shape[1:])
            ns_raw = self._ns_raw(cb)
            x = self.ns_tokenizer(ns_raw)                    # [nb, n_ns, D]
            for l, blk in enumerate(self.blocks):
                at = blk.attn
                h = blk.norm1(x)
                w8 = weights[l] if weights else None
                qkv = (int8_linear(h, w8["ns_qkv"]) if w8
                       else torch.einsum("btk,tnk->btn", h, at.ns_qkv_weight.to(h.dtype)))
                qkv = qkv.view(nb, n_ns, 3, H, dh)
                q, k_n, v_n = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
                if kv_cache:
                    o = cache[l].candidates(q, k_n, v_n).reshape(nb, n_ns, D)
                else:
                    k_s, v_s = cache[l]
                    if at.rotary:                            # the last n_ns of n_s + n_ns tokens
                        q, _ = at.norm_rope(q, None, k_s.shape[1] + n_ns)
                        k_n, _ = qk_norm_rope(k_n, None, at.k_norm.weight, None, at.rope(k_s.shape[1] + n_ns, x.device),
                                              torch.arange(k_s.shape[1], k_s.shape[1] + n_ns, device=x.device),
                                              eps=at.k_norm.eps)
                    k = torch.cat([k_s.expand(nb, -1, -1, -1).to(k_n.dtype), k_n], dim=1)
                    v = torch.cat([v_s.expand(nb, -1, -1, -1).to(v_n.dtype), v_n], dim=1)
                    o = pyramid_attention(q, k, v, impl="mask").reshape(nb, n_ns, D)
                if w8:
                    z = int8_linear(o, w8["out"], residual=x.to(o.dtype))
                    f = int8_linear(blk.norm2(z), w8["ns_w1"], act="gelu")
                    x = int8_linear(f, w8["ns_w2"], residual=z.to(f.dtype))
                    continue
                z = at.out_proj(o) + x
                y = blk.norm2(z)
                f = torch.einsum("btk,tnk->btn", y, blk.ffn.ns_w1.to(y.dtype))
                f = torch.einsum("btk,tnk->btn", F.gelu(f), blk.ffn.ns_w2.to(y.dtype))
                x = z + f
            x = self.final_norm(x)
            hh = self.head_proj(x.reshape(nb, -1))
            scores.append(self.heads[task](hh).squeeze(-1).float())
        for pages in cache if kv_cache else ():
            pages.cache.check_errors()
        if weights and not (xs.is_cuda and torch.cuda.is_current_stream_capturing()):    # a graph's launches are read later
            int8.check_errors(xs.device)
        return torch.cat(scores)

    def _ns_raw(self, batch: dict[str, torch.Tensor]) -> torch.Tensor:
        """The NS tokenizer input of a batch: scalar embeddings + dense features."""
        f2k = self.config.feature_to_batch_key()
        fc = self.config.feature
        feats = {f: batch[f2k.get(f, f)] for f in fc.scalar_feature_names if f2k.get(f, f) in batch}
        scal = self.emb.lookup_groups(feats, [list(fc.scalar_feature_names)], dtype=self._compute_dtype(batch))[0]
        parts = [scal]
        for df in fc.dense_features:
            xd = batch[df.name]
            parts.append(self.dense_projs[df.name](xd) if df.name in self.dense_projs else xd.to(scal.dtype))
        return torch.cat([p.to(scal.dtype) for p in parts], dim=-1)

    def forward_with_cross_scores(self, batch: dict[str, torch.Tensor], cross_task: str = ""):
        h, s_repr, scal = self._backbone(batch)
        preds = {t: head(h).squeeze(-1) for t, head in self.heads.items()}
        user = self.contrastive_user_proj(s_repr.to(h.dtype))
        E = self.config.model.embedding_dim
        names = self.config.feature.scalar_feature_names
        cols = []
        for f in self._item_scalar_names:
            i = names.index(f)
            cols.append(scal[:, i * E:(i + 1) * E])
        item = self.contrastive_item_proj(torch.cat(cols, dim=-1))
        return preds, user @ item.t()
