"""Shared test plumbing: the ``gpu`` marker, fixture loading, tolerances."""

from __future__ import annotations

import sys
from multiprocessing.context import SpawnContext
from pathlib import Path

import numpy as np
import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
GOLDEN = Path(__file__).resolve().parent / "golden"
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

# Tolerance of 16-bit results against the fp32 oracle (the bar the hot path is held to).
BF16_TOL = dict(rtol=2e-2, atol=2e-2)
# fp32 kernels against the oracle.
FP32_TOL = dict(rtol=1e-4, atol=1e-5)
LOSS_REL = 1e-3


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on the B200 box)")


def pytest_collection_modifyitems(config, items):
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


def _share_by_name(target, *args, **kwargs):
    torch.multiprocessing.set_sharing_strategy("file_system")
    target(*args, **kwargs)


class _Rank(SpawnContext.Process):
    def __init__(self, group=None, target=None, name=None, args=(), **more):
        super().__init__(group, _share_by_name, name, (target, *args), **more)


_SPAWNING = ("test_sharded_adamw_cpu", "test_gpu_sharded_adamw", "test_vocab_parallel_cpu", "test_gpu_vocab_parallel")


@pytest.fixture(autouse=True)
def _tensors_outlive_their_process(request, monkeypatch):
    """Spawned ranks hand tensors to the test through a queue and exit.  By default the receiver fetches a
    tensor's file descriptor from its sender, which fails if that is gone by then (a rank ends a few
    milliseconds after its ``put``); shared by name they stay until they have been received.  Only for the
    modules that spawn ranks."""
    if request.module.__name__.endswith(_SPAWNING):
        monkeypatch.setattr(SpawnContext, "Process", _Rank)


def load_golden(name: str):
    return np.load(GOLDEN / name, allow_pickle=False)


@pytest.fixture(scope="session")
def lib():
    from bastile_b200 import _lib

    return _lib.get_lib()


def to_np(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy()


def assert_close(actual, expected, rtol, atol, what=""):
    a = to_np(actual) if isinstance(actual, torch.Tensor) else np.asarray(actual, np.float32)
    e = to_np(expected) if isinstance(expected, torch.Tensor) else np.asarray(expected, np.float32)
    assert a.shape == e.shape, f"{what}: shape {a.shape} vs {e.shape}"
    assert np.isfinite(a).all(), f"{what}: non-finite values"
    err = np.abs(a - e)
    bound = atol + rtol * np.abs(e)
    bad = err > bound
    if bad.any():
        i = np.unravel_index(np.argmax(err - bound), err.shape)
        raise AssertionError(
            f"{what}: {int(bad.sum())}/{bad.size} elements off; worst at {i}: got {a[i]!r}, want {e[i]!r} "
            f"(|err| {err[i]:.3e} > {bound[i]:.3e})"
        )
