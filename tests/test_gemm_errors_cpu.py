"""A GEMM that gave up, as the trainer sees it (the error word is a stub: no kernel runs)."""
import importlib
from pathlib import Path

import pytest
import torch

from primus_dlrm_b200.ops import dense

ROOT = Path(__file__).resolve().parent.parent


def _trainer(tmp_path, steps, log_interval):
    from primus_dlrm_b200.config import Config
    from primus_dlrm_b200.data.synthetic import generate_batch
    from primus_dlrm_b200.models.onetrans import OneTransModel
    from primus_dlrm_b200.training.engine import TrainEngine
    trainer = importlib.import_module("primus_dlrm_b200.training.trainer")
    cfg = Config.load(str(ROOT / "configs" / "onetrans_tiny.yaml"))
    cfg.data.history_length = 4
    cfg.train.batch_size, cfg.train.kernels = 4, "eager"
    cfg.train.epochs, cfg.train.save_checkpoint = 1, True
    model = OneTransModel(cfg)
    eng = TrainEngine(model, cfg, torch.device("cpu"), total_steps=steps)
    return eng, trainer.DistributedTrainer(model, eng, [generate_batch(cfg, 4, seed=i) for i in range(steps)], cfg,
                                           torch.device("cpu"), log_interval=log_interval, run_dir=tmp_path)


@pytest.mark.parametrize("fails_at,log_interval,seen_at", [(2, 2, 3), (3, 100, 4)])
def test_training_stops_at_the_next_look(fails_at, log_interval, seen_at, tmp_path, monkeypatch):
    """At a log step, else at the epoch's end and before its checkpoint."""
    eng, tr = _trainer(tmp_path, 4, log_interval)
    word = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(dense, "_err", lambda device: word)
    monkeypatch.setattr(dense._ext, "native_enabled", lambda device=None: True)
    monkeypatch.setattr(dense, "gemm_error_code", lambda device: int(word.item()))
    step = eng.step

    def failing(batch):
        out = step(batch)
        if eng.global_step == fails_at:
            word.fill_(2)
        return out

    # the kernels stay those of the CPU: only the word is asked as on a GPU
    monkeypatch.setattr(eng, "step", failing)
    with pytest.raises(RuntimeError, match="GEMM: a bounded wait"):
        tr.train()
    assert eng.global_step == seen_at and not list(tmp_path.rglob("*.pt"))
    assert word.item() == 0                                  # raised once


def test_training_stops_where_the_attention_gave_up(tmp_path, monkeypatch):
    from primus_dlrm_b200.ops import attention
    eng, tr = _trainer(tmp_path, 2, 1)
    word = torch.full((1,), 2, dtype=torch.int32)
    monkeypatch.setattr(attention, "_err_word", lambda device: word)
    monkeypatch.setattr(attention, "attention_error_code", lambda device: int(word.item()))
    monkeypatch.setattr(attention._ext, "native_enabled", lambda device=None: True)
    monkeypatch.setattr(dense, "gemm_error_code", lambda device: 0)
    with pytest.raises(RuntimeError, match="attention: a bounded wait"):
        tr.train()
    assert eng.global_step == 1 and word.item() == 0


def test_training_without_errors_runs_and_saves(tmp_path):
    eng, tr = _trainer(tmp_path, 3, 1)
    tr.train()
    assert eng.global_step == 3 and list(tmp_path.rglob("*.pt"))
