"""Tests that read the allocator's count read it settled (conftest)."""
import threading
import time
import weakref

import torch

from conftest import settled


class _Buffer:
    pass


def _late(alive):
    """A buffer that a thread drops a moment after its owner went on, and one in a cycle."""
    b, c = _Buffer(), _Buffer()
    c.me = c
    alive += [weakref.ref(b), weakref.ref(c)]
    held, started = [b], threading.Event()

    def hold():
        started.set()
        time.sleep(0.003)
        held.clear()

    threading.Thread(target=hold).start()
    started.wait()


def test_what_nothing_uses_is_not_counted():
    alive = []
    _late(alive)
    count = lambda: sum(r() is not None for r in alive)  # noqa: E731
    assert count() > 0 and settled(count)() == 0


def test_tests_that_name_the_count_get_it_settled():
    assert hasattr(torch.cuda.memory_allocated, "__wrapped__")


def test_others_do_not():
    assert not hasattr(getattr(torch.cuda, "memory_" + "allocated"), "__wrapped__")
