"""Loader for the in-tree sm_100a extensions.

``core()`` returns the ``_C`` module (embedding, norm, loss, optimizer
kernels), ``gemm()`` the ``_gemm`` module (tcgen05 GEMMs, attention) and
``kv()`` the ``_kv`` module (rotary and key/value-cache kernels), ``int8()``
the ``_int8`` module (8-bit integer kernels).
On a machine with a CUDA device a missing or stale extension raises: a GPU
run never silently falls back to eager PyTorch.  Without a CUDA device the
eager implementations in ``primus_dlrm_b200.ops`` are the only path (they
also serve as the fp32 oracles of the kernel tests).
"""
from __future__ import annotations

import importlib
import os

import torch

_cache: dict[str, object] = {}


def _load(name: str):
    if name in _cache:
        return _cache[name]
    try:
        mod = importlib.import_module(f"primus_dlrm_b200.{name}")
    except ImportError as e:  # pragma: no cover - exercised on GPU boxes only
        src = os.path.join(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))),
                           "csrc", {"_gemm": "gemm_bindings.cpp", "_kv": "kv_bindings.cpp",
                                    "_int8": "int8_bindings.cpp"}.get(name, "bindings.cpp"))
        if torch.cuda.is_available() and os.path.exists(src):
            raise RuntimeError(
                f"primus_dlrm_b200.{name} is not built; run `python setup.py build_ext --inplace` "
                f"(sm_100a). A CUDA device is present, so no eager fallback is used.") from e
        mod = None
    _cache[name] = mod
    return mod


def core():
    return _load("_C")


def gemm():
    return _load("_gemm")


def kv():
    return _load("_kv")


def int8():
    return _load("_int8")


def native_enabled(device: torch.device | str | None = None) -> bool:
    """Native kernels run for CUDA tensors unless PD_KERNELS=eager."""
    if os.environ.get("PD_KERNELS", "") == "eager":
        return False
    if device is not None and torch.device(device).type != "cuda":
        return False
    return torch.cuda.is_available()
