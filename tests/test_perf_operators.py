"""The calls that perf/operators.py makes as a user: on the stream and device that are current at the call.  No GPU."""
import importlib.util
import os
import types

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def ops():
    spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(ROOT, "perf", "operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_a_call_goes_to_the_stream_that_is_current(ops, monkeypatch):
    import moeflux_b200

    opened, now = [], types.SimpleNamespace(device_index=0, cuda_stream=0)

    class FakeCtx:
        def __init__(self, **fields):
            opened.append(self)
            self.device, self.stream = fields.get("device", 0), "its own"

        def set_stream(self, stream):
            self.stream = stream

    monkeypatch.setattr(moeflux_b200, "Ctx", FakeCtx)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: now)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now.device_index)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: now.cuda_stream, raising=False)
    for device, stream in [(0, 0), (0, 7), (1, 0), (0, 7), (0, 0), (1, 9)]:
        now.device_index, now.cuda_stream = device, stream
        c = ops._handle()
        assert (c.device, c.stream) == (device, stream)
    assert len(opened) == 4  # kept, and not opened again
