"""OneTrans trained with its activations in 8 bits, and scored with its weights as 8-bit integers."""
import pytest
import torch
import torch.nn.functional as F

from primus_dlrm_b200.evaluation.metrics import score_candidates, serving_weights
from primus_dlrm_b200.models import onetrans
from primus_dlrm_b200.models.onetrans import OneTransModel
from primus_dlrm_b200.ops.int8 import Int8Weight
from test_models_cpu import _batch, _config
from test_onetrans_rotary import _model, _split


def _pair(device, **transformer):
    """The same model with activations in 16 and in 8 bits."""
    a, b = (_model(device, activation_bits=n, **transformer) for n in (16, 8))
    b.load_state_dict(a.state_dict())
    return a.train(), b.train()


def _step(model, batch, autocast=False):
    model.zero_grad()
    with torch.autocast(next(iter(batch.values())).device.type, dtype=torch.bfloat16, enabled=autocast):
        total, _, logits = model.forward_loss(batch, {"listen_plus": 1.0}, [])
    total.backward()
    return total.item(), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None and n.startswith("blocks")}


# A saved value is off by at most 2^-7 of its block's largest magnitude, and by 2^-8.8 of it on average; the largest of 32
# normal values is about 2.5 times their size. So each block's gradients are off by some 0.6 %, those of the first blocks by
# the sum over the blocks above: 0.05 leaves a factor of four for these models of up to four blocks.
OFF = 0.05


@pytest.mark.parametrize("transformer", [dict(dropout=0.0), dict(dropout=0.0, rotary=True), dict(dropout=0.0, use_pyramid=False),
                                         dict(dropout=0.0, d_model=40)])
def test_training_with_activations_in_8_bits(transformer):
    a, b = _pair("cpu", **transformer)
    batch = _batch(B=6, windows=2)
    (la, ga), (lb, gb) = _step(a, batch), _step(b, batch)
    assert abs(la - lb) < 1e-6 and ga.keys() == gb.keys()
    assert any(not torch.equal(ga[n], gb[n]) for n in ga)
    for n in ga:
        assert (ga[n] - gb[n]).norm() <= OFF * ga[n].norm() + 1e-7, n


def test_training_with_dropout_runs():
    _, b = _pair("cpu", dropout=0.3)
    loss, grads = _step(b, _batch(B=4, windows=2))
    assert loss == loss and all(g.isfinite().all() for g in grads.values())


def test_bits_are_checked():
    cfg = _config("onetrans", windows=2)
    assert cfg.model.transformer.activation_bits == 16
    cfg.model.transformer.activation_bits = 4
    with pytest.raises(ValueError, match="activation_bits"):
        OneTransModel(cfg)


@pytest.mark.parametrize("kv_cache", [None, "fp8"])
@pytest.mark.parametrize("rotary", [True, False])
def test_scoring_uses_every_weight(rotary, kv_cache, monkeypatch):
    """With the integer product replaced by the exact one the scores are those of the plain path."""
    model = _model(rotary=rotary)
    user, cand, _ = _split(_batch(B=7, L=30, windows=2, seed=5), 7)

    def exact(x, w, bias=None, act=None, residual=None):
        y = torch.einsum("btk,tnk->btn", x, w) if w.dim() == 3 else x @ w.t()
        y = F.gelu(y) if act == "gelu" else y
        return y if residual is None else y + residual

    ref = model.score_candidates(user, cand, "listen_plus", batch_size=3, kv_cache=kv_cache)
    monkeypatch.setattr(Int8Weight, "from_float", classmethod(lambda cls, w: w))
    monkeypatch.setattr(onetrans, "int8_linear", exact)
    got = score_candidates(model, user, cand, "listen_plus", 3, kv_cache, weights=serving_weights(model, "int8"))
    torch.testing.assert_close(got, ref, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("kv_cache", [None, "fp8"])
def test_scores_of_integer_weights(kv_cache):
    """Weights and activations are off by at most half of 1/127 of a channel's or token's largest magnitude; the scores'
    differences stay small against their spread, and do not depend on how candidates are batched."""
    model = _model(rotary=True)
    user, cand, _ = _split(_batch(B=40, L=30, windows=2, seed=5), 40)
    w8 = model.int8_weights()
    ref = model.score_candidates(user, cand, "listen_plus", kv_cache=kv_cache)
    got = model.score_candidates(user, cand, "listen_plus", kv_cache=kv_cache, weights=w8)
    assert not torch.equal(ref, got) and (ref - got).norm() <= 0.1 * (ref - ref.mean()).norm()
    again = model.score_candidates(user, cand, "listen_plus", batch_size=7, kv_cache=kv_cache, weights=w8)
    torch.testing.assert_close(got, again, rtol=1e-4, atol=1e-5)
    with pytest.raises(ValueError, match="blocks"):
        model.score_candidates(user, cand, "listen_plus", weights=w8[:1])
    with pytest.raises(ValueError, match="int4"):
        serving_weights(model, "int4")


def test_models_without_integer_weights_say_so():
    from primus_dlrm_b200.parallel.build import build_model
    model = build_model(_config("dlrm"), device=torch.device("cpu"))
    with pytest.raises(ValueError, match="OneTrans"):
        serving_weights(model, "int8")
    with pytest.raises(ValueError, match="its own"):
        score_candidates(model, {}, {}, "listen_plus", weights=[])


def test_ranking_with_integer_weights():
    from pathlib import Path

    from primus_dlrm_b200.config import Config
    from primus_dlrm_b200.data.dataset import SyntheticEvalDataset
    from primus_dlrm_b200.evaluation.metrics import evaluate_ranking, evaluate_ranking_peruser
    cfg = Config.load(str(Path(__file__).resolve().parent.parent / "configs" / "onetrans_tiny.yaml"))
    model = OneTransModel(cfg).eval()
    ds = SyntheticEvalDataset(cfg, num_users=3, num_items_with_history=50)
    for res in (evaluate_ranking(model, ds, torch.device("cpu"), candidate_item_ids=torch.arange(40).numpy(), ks=[5, 10],
                                 weights="int8"),
                evaluate_ranking_peruser(model, ds, torch.device("cpu"), ks=[5, 10], top_n=20, weights="int8")):
        assert all(0.0 <= v <= 1.0 for v in res.values() if isinstance(v, float)) and "ndcg@10" in res
    with pytest.raises(ValueError, match="int4"):
        evaluate_ranking(model, ds, torch.device("cpu"), ks=[5], weights="int4")


@pytest.mark.gpu
@pytest.mark.parametrize("transformer", [dict(), dict(rotary=True), dict(d_model=128, heads=4), dict(attention_impl="sdpa")])
def test_gpu_training_with_activations_in_8_bits(transformer):
    kw = {"dropout": 0.0, "attention_impl": "fav4", **transformer}
    a, b = _pair("cuda", **kw)
    batch = {k: v.cuda() for k, v in _batch(B=32, windows=2).items()}
    (la, ga), (lb, gb) = _step(a, batch, True), _step(b, batch, True)
    # the loss kernel adds its rows' 32 terms by atomics, in any order: 31 additions of at most 2^-24 of the sum each
    assert abs(la - lb) <= 31 * 2.0 ** -24 * abs(la) and ga.keys() == gb.keys()
    for n in ga:
        # and the roundings of bf16 on the way, which the two backward passes take at other places
        assert (ga[n] - gb[n]).norm() <= (OFF + 2 ** -6) * ga[n].norm() + 1e-7, n


@pytest.mark.gpu
def test_gpu_training_holds_less_memory():
    a, b = _pair("cuda", dropout=0.0, attention_impl="fav4", d_model=256, heads=8)
    batch = {k: v.cuda() for k, v in _batch(B=256, windows=2).items()}
    held = []
    for m in (a, b):
        kept = {}

        def keep(t):
            kept[t.data_ptr()] = max(kept.get(t.data_ptr(), 0), t.numel() * t.element_size())
            return t

        with torch.autocast("cuda", dtype=torch.bfloat16), torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
            total, _, _ = m.forward_loss(batch, {"listen_plus": 1.0}, [])
        held.append(sum(kept.values()))
        del total, kept
    # x, GELU and GELU' in bf16 against x and the pre-activation in 33 / 32 bytes, and the QKV projection's input
    D, F_, ns, kv, saved = 256, 512, 4, 30 + 4, 0
    for q in onetrans.pyramid_schedule(30, ns, len(a.blocks)):
        saved += (q + ns) * (2 * D + 4 * F_ - (D + F_) * 33 // 32) + kv * (2 * D - D * 33 // 32)
        kv = q + ns
    assert held[0] - held[1] == 256 * saved, (held, 256 * saved)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_cache", [None, "fp8"])
@pytest.mark.parametrize("autocast", [True, False])
def test_gpu_scores_of_integer_weights(autocast, kv_cache, monkeypatch):
    """The kernels in the model, against the same integers in PyTorch; what differs are roundings of bf16 (2^-8), which
    two layers and the head may amplify by 16 at most here."""
    from primus_dlrm_b200.ops.int8 import _linear_ref
    model = _model("cuda", rotary=True, attention_impl="fav4")
    user, cand, _ = _split({k: v.cuda() for k, v in _batch(B=70, L=40, windows=2, seed=5).items()}, 70)
    w8 = model.int8_weights()

    def run():
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            return model.score_candidates(user, cand, "listen_plus", batch_size=32, kv_cache=kv_cache, weights=w8)

    got = run()
    plain = lambda x, w, bias=None, act=None, residual=None: _linear_ref(x, w, bias, act, residual)  # noqa: E731
    monkeypatch.setattr(onetrans, "int8_linear", plain)
    with torch.autocast("cuda", enabled=False):
        ref = run()
    assert (got - ref).abs().max().item() <= 2 ** -4 * ref.abs().max().item()
