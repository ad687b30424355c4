"""Activations in 8 bits and integer weights where the dense parameters are averaged or sharded (gloo, 2 ranks)."""
import copy
import functools

import pytest
import torch

import test_distributed_cpu as base
from dist_utils import run_ranks


def _config(dense, opt="sgd"):
    cfg = base_config(dense, opt)
    cfg.model.transformer.activation_bits = 8
    return cfg


base_config = base._config


def _train_worker(rank, world, dense, opt, steps):
    base._config = _config
    return base._dist_worker(rank, world, dense, opt, steps)


@pytest.mark.parametrize("dense,opt,tab_atol", [("ddp", "sgd", 1e-6), ("fsdp", "adam", 5e-4), ("zero2", "adam", 5e-4)])
def test_training_matches_single_process(dense, opt, tab_atol, monkeypatch):
    """As the 16-bit model's (the codes are of the rows' values, which do not depend on the ranks): losses and weights after
    two steps, and they are not the 16-bit model's."""
    res = run_ranks(_train_worker, 2, dense, opt, 2)
    _, sixteen = base._oracle(dense, opt, 2)
    monkeypatch.setattr(base, "_config", _config)
    ref_losses, ref_sd = base._oracle(dense, opt, 2)
    losses, sd = res[0]
    assert losses == pytest.approx(ref_losses, rel=1e-4, abs=1e-5) and set(sd) == set(ref_sd)
    for k in ref_sd:
        atol = tab_atol if ".embeddings." in k else 5e-5
        torch.testing.assert_close(sd[k], ref_sd[k], rtol=1e-3, atol=atol, msg=lambda m: f"{k}: {m}")
    assert any(not torch.equal(ref_sd[k], sixteen[k]) for k in ref_sd if k.startswith("blocks"))


def _setup(world):
    from primus_dlrm_b200.data.synthetic import generate_batch
    from primus_dlrm_b200.parallel.build import build_model
    cfg = base_config("fsdp", "adam")
    torch.manual_seed(0)
    model = build_model(cfg).eval()
    return cfg, model, base._user_cand(cfg, generate_batch(cfg, 6, seed=7))


def _score_worker(rank, world):
    from primus_dlrm_b200.evaluation.metrics import score_candidates, serving_weights
    from primus_dlrm_b200.parallel.build import build_model
    from primus_dlrm_b200.parallel.fsdp import DTensor
    from primus_dlrm_b200.parallel.state import load_full_state_dict
    from primus_dlrm_b200.parallel.wrapper import wrap_model
    cfg, ref, (user, cand) = _setup(world)
    full = copy.deepcopy(ref.state_dict())
    model, _ = wrap_model(build_model(cfg, meta_device=True), torch.device("cpu"), cfg)
    load_full_state_dict(model, full)
    model.eval()
    w8 = serving_weights(model, "int8")
    assert isinstance(model.blocks[0].attn.ns_qkv_weight, DTensor)     # sharded again, the integers stay whole
    assert type(w8[0]["ns_qkv"].codes) is torch.Tensor and w8[0]["ns_qkv"].codes.shape == ref.blocks[0].attn.ns_qkv_weight.shape
    score = functools.partial(score_candidates, model, user, cand, "listen_plus", weights=w8)
    return score(), score(batch_size=4)


def test_integer_weights_of_sharded_parameters():
    from primus_dlrm_b200.evaluation.metrics import score_candidates, serving_weights
    res = run_ranks(_score_worker, 2)
    _, ref, (user, cand) = _setup(2)
    want = score_candidates(ref, user, cand, "listen_plus", weights=serving_weights(ref, "int8"))
    assert not torch.equal(want, score_candidates(ref, user, cand, "listen_plus"))
    for got in res.values():
        for s in got:
            torch.testing.assert_close(s, want, rtol=1e-4, atol=1e-5)
