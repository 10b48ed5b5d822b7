import functools
import gc
import os
import sys
import time

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA (B200, sm_100a) device")
    config.addinivalue_line("markers", "dist: spawns multiple processes")
    config.addinivalue_line("markers", "slow: long-running test")


def pytest_collection_modifyitems(config, items):
    import torch

    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for it in items:
        if "gpu" in it.keywords:
            it.add_marker(skip)


def settled(read):
    """`read` of the allocator's count, once what nothing uses any more is gone: objects that wait for the
    garbage collector, and what a thread of the autograd engine still holds. That thread wakes the caller
    of a backward pass before it drops its own reference to the pass and the gradients in it, and where the
    caller takes its processor the reference outlives the call by milliseconds."""

    @functools.wraps(read)
    def call(*args, **kw):
        time.sleep(0.02)
        gc.collect()
        return read(*args, **kw)

    return call


@pytest.fixture(autouse=True)
def _settled_allocator(request):
    """Tests that name torch.cuda.memory_allocated read it settled."""
    if "memory_allocated" in getattr(getattr(request.function, "__code__", None), "co_names", ()):
        import torch

        patch = request.getfixturevalue("monkeypatch")
        patch.setattr(torch.cuda, "memory_allocated", settled(torch.cuda.memory_allocated))
