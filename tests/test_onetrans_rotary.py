"""OneTrans with query/key norms and rotation, and scoring over the 8-bit paged cache."""
import pytest
import torch

from primus_dlrm_b200.models import onetrans
from primus_dlrm_b200.models.onetrans import OneTransModel
from primus_dlrm_b200.ops.kv_cache import PagedKVCache, paged_attention_ref
from primus_dlrm_b200.ops.rotary import rotate_ref
from test_models_cpu import _batch, _config


def _split(full, n):
    user_keys = [k for k in full if k.startswith("hist_")] + ["uid", "user_counters"]
    user = {k: full[k][:1] for k in user_keys}
    cand = {k: full[k] for k in ("item_id", "artist_id", "album_id", "audio_embed", "item_counters", "cross_counters")}
    rows = dict(cand)
    for k in user_keys:
        rows[k] = user[k].expand(n, *user[k].shape[1:])
    return user, cand, rows


def _model(device="cpu", seed=0, d_model=64, heads=2, **transformer):
    cfg = _config("onetrans", windows=2)
    for k, v in {"d_model": d_model, "n_heads": heads, **transformer}.items():
        setattr(cfg.model.transformer, k, v)
    torch.manual_seed(seed)
    model = OneTransModel(cfg, device=torch.device(device)).eval()
    with torch.no_grad():
        for blk in model.blocks:
            if blk.attn.rotary:
                blk.attn.q_norm.weight.mul_(1.3)
                blk.attn.k_norm.weight.add_(0.1 * torch.randn_like(blk.attn.k_norm.weight))
    return model


def test_off_by_default_and_same_state_dict():
    a, b = _model(), _model(rotary=True)
    new = set(b.state_dict()) - set(a.state_dict())
    assert set(a.state_dict()) <= set(b.state_dict())
    assert new == {f"blocks.{i}.attn.{n}_norm.weight" for i in range(len(a.blocks)) for n in "qk"}


@pytest.mark.parametrize("pyramid", [True, False])
def test_scoring_with_rotation_is_exact(pyramid):
    model = _model(rotary=True, use_pyramid=pyramid, pos_embed=False)
    user, cand, rows = _split(_batch(B=7, windows=2, seed=5), 7)
    with torch.no_grad():
        ref = model(rows)["listen_plus"]
        got = model.score_candidates(user, cand, "listen_plus", batch_size=3)
    torch.testing.assert_close(got, ref, rtol=1e-4, atol=1e-5)


class _WidePages(PagedKVCache):
    """Pages that keep fp32 values: scoring over them must be exact, so what is left is how pages and positions are used."""

    def __init__(self, n_pages, H, d, P, device=None):
        super().__init__(n_pages, H, d, P, device)
        self.wide = [torch.full((n_pages, H, P, d), float("nan")) for _ in range(2)]

    def append(self, k, v, table, lens, *, k_weight=None, norm_eps=None, rope=None):
        for b in range(k.shape[0]):
            x, at = k[b].float(), int(lens[b])
            if norm_eps is not None:
                x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + norm_eps) * k_weight
            if rope is not None:
                x = rotate_ref(x, rope[at:at + x.shape[0]])
            for i in range(x.shape[0]):
                page, row = int(table[b, (at + i) // self.page_size]), (at + i) % self.page_size
                self.wide[0][page, :, row], self.wide[1][page, :, row] = x[i], v[b, i].float()

    def copy_pages(self, src, dst):
        for w in self.wide:
            w[dst] = w[src]

    def attend(self, q, table, lens):
        out = torch.empty_like(q)
        for b in range(q.shape[0]):
            n, T = q.shape[1], int(lens[b])
            k, v = (w[table[b].long()].transpose(1, 2).flatten(0, 1)[:T] for w in self.wide)
            w = torch.einsum("ihd,jhd->hij", q[b], k) * q.shape[-1] ** -0.5
            w = w.masked_fill(torch.arange(T) > (T - n + torch.arange(n))[:, None], float("-inf"))
            out[b] = torch.einsum("hij,jhd->ihd", w.softmax(-1), v)
        return out


@pytest.mark.parametrize("rotary", [True, False])
@pytest.mark.parametrize("L", [10, 21, 30, 64])
def test_pages_and_positions(rotary, L, monkeypatch):
    """Histories that end inside a page, at its end, and candidates that spill into the next one."""
    model = _model(rotary=rotary)
    user, cand, rows = _split(_batch(B=7, L=L, windows=2, seed=5), 7)
    with torch.no_grad():
        ref = model.score_candidates(user, cand, "listen_plus")
        monkeypatch.setattr(onetrans, "PagedKVCache", _WidePages)
        monkeypatch.setattr(onetrans, "paged_attention", lambda q, c, t, n, max_len=None: c.attend(q, t, n))
        for size in (3, 7):
            got = model.score_candidates(user, cand, "listen_plus", batch_size=size, kv_cache="fp8")
            torch.testing.assert_close(got, ref, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("rotary", [True, False])
def test_scoring_over_8_bit_pages(rotary):
    """The result does not depend on how candidates are batched."""
    model = _model(rotary=rotary)
    user, cand, rows = _split(_batch(B=7, L=30, windows=2, seed=5), 7)
    with torch.no_grad():
        got = model.score_candidates(user, cand, "listen_plus", batch_size=3, kv_cache="fp8")
        again = model.score_candidates(user, cand, "listen_plus", batch_size=7, kv_cache="fp8")
    torch.testing.assert_close(got, again, rtol=1e-4, atol=1e-5)
    assert not torch.equal(got, model.score_candidates(user, cand, "listen_plus"))
    with pytest.raises(ValueError):
        model.score_candidates(user, cand, "listen_plus", kv_cache="int4")


def test_training_step_moves_the_norms():
    model = _model(rotary=True).train()
    batch = _batch(B=4, windows=2)
    total, _, _ = model.forward_loss(batch, {"listen_plus": 1.0}, [])
    total.backward()
    for blk in model.blocks:
        for w in (blk.attn.q_norm.weight, blk.attn.k_norm.weight):
            assert w.grad is not None and torch.isfinite(w.grad).all() and w.grad.abs().max() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("impl", ["fav4", "sdpa"])
def test_gpu_training_step_matches_cpu(impl):
    """bf16 autocast on the GPU against fp32 on the CPU: loss and gradients of the norms."""
    gpu, cpu = _model("cuda", rotary=True, attention_impl=impl), _model(rotary=True, attention_impl=impl)
    cpu.load_state_dict({k: v.cpu() for k, v in gpu.state_dict().items()})
    batch = _batch(B=32, windows=2)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        total, _, _ = gpu.forward_loss({k: v.cuda() for k, v in batch.items()}, {"listen_plus": 1.0}, [])
    total.backward()
    want, _, _ = cpu.forward_loss(batch, {"listen_plus": 1.0}, [])
    want.backward()
    assert abs(total.item() - want.item()) < 2e-2
    for a, b in zip(gpu.blocks, cpu.blocks):
        for x, y in ((a.attn.q_norm, b.attn.q_norm), (a.attn.k_norm, b.attn.k_norm)):
            x, y = x.weight.grad.cpu(), y.weight.grad
            assert (x - y).norm() <= 0.25 * y.norm() + 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [True, False])
def test_gpu_scoring_over_8_bit_pages(rotary, monkeypatch):
    """The three operators together, against the same pages with plain attention in 32 bits: what differs are roundings
    of bf16 (2^-8), which two layers and the head may amplify by 16 at most here."""
    model = _model("cuda", rotary=rotary, attention_impl="fav4")
    user, cand, _ = _split({k: v.cuda() for k, v in _batch(B=70, L=40, windows=2, seed=5).items()}, 70)

    def run():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            a = model.score_candidates(user, cand, "listen_plus", batch_size=32, kv_cache="fp8")
        return a, model.score_candidates(user, cand, "listen_plus", kv_cache="fp8")     # fp32 outside autocast

    got = run()
    monkeypatch.setattr(onetrans, "paged_attention",
                        lambda q, c, t, n, max_len=None: paged_attention_ref(q, c, t, n)[0].to(q.dtype))
    for a, b in zip(got, run()):
        assert (a - b).abs().max().item() <= 2 ** -4 * b.abs().max().item()
