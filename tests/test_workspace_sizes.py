"""CPU: scratch sizes that follow from a device's number of SMs are asked for on that device, once each."""

import contextlib

import pytest
import torch

from hyper_multicore_b200 import _lib, kernels as K


class _Machine:
    """Two devices of 100 and 148 SMs; the library answers for the current one, as the real one does."""

    def __init__(self):
        self.current, self.sms, self.calls = 0, (100, 148), 0

    def hmc_row_norm_grad_workspace_bytes(self, rows, hidden):
        self.calls += 1
        return self.sms[self.current] * rows * hidden

    @contextlib.contextmanager
    def guard(self, index):
        before, self.current = self.current, index
        yield
        self.current = before


@pytest.fixture
def machine(monkeypatch):
    fake = _Machine()
    monkeypatch.setattr(_lib, "load", lambda: fake)
    monkeypatch.setattr(torch.cuda, "device", fake.guard)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: fake.current)
    K._size_on.cache_clear()
    yield fake
    K._size_on.cache_clear()


def test_a_size_is_that_of_the_tensors_device(machine):
    name = "hmc_row_norm_grad_workspace_bytes"
    first, second = torch.device("cuda", 0), torch.device("cuda", 1)
    assert K._size(name, 3, 5, device=second) == 148 * 15 and machine.current == 0
    assert K._size(name, 3, 5, device=first) == 100 * 15
    assert K._size(name, 3, 5) == 100 * 15  # the current device
    machine.current = 1
    assert K._size(name, 3, 5) == 148 * 15 and K._size(name, 3, 5, device=first) == 100 * 15
    assert machine.calls == 2
    assert K._size(name, 3, 6, device=first) == 100 * 18 and machine.calls == 3
