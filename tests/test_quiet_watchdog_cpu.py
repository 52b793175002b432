"""Before a capture the trainer waits until the process group's watchdog has seen every eager collective done -- with an nccl
group that reduces gradients, and only then."""
import time
import types

import pytest
import torch

from dphubert_amd.trainer import Trainer


@pytest.mark.parametrize("enabled,backend,waits", [(True, "nccl", True), (True, "gloo", False), (False, "nccl", False)])
def test_waits_for_the_device_and_then_for_the_watchdog(monkeypatch, enabled, backend, waits):
    done = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: done.append("device"))
    monkeypatch.setattr(time, "sleep", lambda s: done.append(s))
    me = types.SimpleNamespace(reducer=types.SimpleNamespace(enabled=enabled, backend=backend),
                               WATCHDOG_QUIET_S=Trainer.WATCHDOG_QUIET_S)
    Trainer._quiet_watchdog(me)
    # (it looks every 0.1 s: three looks)
    assert done == (["device", Trainer.WATCHDOG_QUIET_S] if waits else []) and Trainer.WATCHDOG_QUIET_S >= 0.3
