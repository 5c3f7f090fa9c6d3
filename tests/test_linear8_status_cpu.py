"""The status word that calls on a device share: made once whichever thread comes first (torch's device calls are stood in for)."""
import contextlib
import threading
import time
import types

import pytest
import torch

from vllm_tgis_adapter_b200.engine import linear8


@pytest.fixture
def no_device(monkeypatch):
    """What with_status asks of a device, answered without one, and slowly."""
    made = []

    def zeros(*shape, **kw):
        time.sleep(0.02)
        made.append(real(*shape, **kw))
        time.sleep(0.02)
        return made[-1]

    real = torch.zeros
    monkeypatch.setattr(torch, "zeros", zeros)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: types.SimpleNamespace(synchronize=lambda: time.sleep(0.02)))
    return made


def at_once(n, work):
    start, got = threading.Barrier(n), [None] * n

    def run(i):
        start.wait()
        got[i] = work()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return got


def test_threads_that_come_first_together_share_one_word(no_device):
    on = linear8._Device(torch.device("cpu"))
    got = at_once(8, lambda: on.with_status().status_at)
    assert len(no_device) == 1 and got == [no_device[0].data_ptr()] * 8


def test_threads_that_come_first_together_share_one_device(monkeypatch):
    class Slow(linear8._Device):
        def __init__(self, device):
            time.sleep(0.02)
            super().__init__(device)

    monkeypatch.setattr(linear8, "_Device", Slow)
    monkeypatch.setattr(linear8, "_devices", {})
    got = at_once(8, lambda: linear8._of(torch.device("cpu")))
    assert all(on is got[0] for on in got)


def test_a_stall_is_counted_once_and_told_to_all(no_device):
    on = linear8._Device(torch.device("cpu")).with_status()
    layers = [linear8._Checked() for _ in range(6)]
    for layer in layers:
        layer._watch(on)
    on.status.fill_(1)
    told = []

    def check(layer):
        try:
            layer.check()
        except RuntimeError:
            told.append(layer)

    todo = list(layers)
    at_once(6, lambda: check(todo.pop()))
    assert on.stalls == 1 and len(told) == 6 and int(on.status) == 0
    at_once(6, lambda: [check(layer) for layer in layers])
    assert len(told) == 6
