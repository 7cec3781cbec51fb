"""Transport.quiesce leaves nothing for the process group's watchdog thread to poll while a step is recorded."""
from types import SimpleNamespace

import torch


def test_quiesce_waits_for_the_device_then_for_the_watchdogs_list(monkeypatch):
    from ocean.parallel import Transport
    calls = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: calls.append("device"))
    t = Transport.__new__(Transport)
    t.group = SimpleNamespace(_wait_for_pending_works=lambda: calls.append("list"))
    t.backend = "nccl"
    t.quiesce()
    assert calls == ["device", "list"]                       # a collective leaves the list only once it has completed
    t.backend = "gloo"
    t.quiesce()
    assert calls == ["device", "list"]


def test_the_process_group_offers_the_wait():
    from torch._C._distributed_c10d import ProcessGroup
    assert callable(ProcessGroup._wait_for_pending_works)
