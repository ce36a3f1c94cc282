"""pytest configuration: the `gpu` marker and shared fixtures.

Tests marked ``gpu`` need a CUDA device and the built ``libbm_layer_ops.so``;
they fail (not skip) without them, so a GPU run can never pass on a fallback.
Everything else runs on a CPU-only machine.
"""
import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if REPO not in sys.path:
    sys.path.insert(0, REPO)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200) and the built sm_100a library")


# These need programs built from the reference's own sources and fail where it is absent.
NEED_THE_REFERENCE = ("test_gpu_engine.py", "test_gpu_reference.py")


def pytest_collection_modifyitems(items):
    """They run after all others, so that a run that stops at its first failure (-x) has run
    everything that needs no reference."""
    items.sort(key=lambda item: item.path.name in NEED_THE_REFERENCE)


@pytest.fixture(scope="session")
def cuda():
    import torch

    assert torch.cuda.is_available(), "gpu tests need a CUDA device"
    from baremetalinferenceengine_b200 import load

    load()  # raises if the library is missing: no fallback
    return torch.device("cuda", 0)
