"""Calls on tensors of a device that is not the current one: the C entries set up and launch kernels on the current
device, and a stream handle alone does not name one (every device's default stream has the handle 0)."""
import re
from pathlib import Path

import pytest
import torch

from vmonarch_b200 import _native as N


@pytest.fixture
def devices(monkeypatch):
    """Two devices that are not there; returns a function that tells the current one."""
    now = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.before

    monkeypatch.setattr(N, "current_device", lambda: now[0])
    monkeypatch.setattr(N, "raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    return lambda: now[0]


@pytest.mark.parametrize("index", [0, 1, None])
def test_launch_makes_the_tensors_device_current(devices, index):
    seen = []
    N.launch("vmb_test", lambda *a: seen.append((devices(), a)) or 0, torch.device("cuda", index) if index is not None
             else torch.device("cuda"), "x", 3)
    assert seen == [(index or 0, ("x", 3, 100 + (index or 0)))] and devices() == 0


@pytest.mark.parametrize("index", [0, 1])
def test_launch_reports_errors_and_leaves_the_device_as_it_was(devices, index):
    with pytest.raises(N.VMonarchError, match="vmb_test failed"):
        N.launch("vmb_test", lambda *a: 1, torch.device("cuda", index))
    assert devices() == 0

    def stop(*_):
        raise KeyError
    with pytest.raises(KeyError):
        N.launch("vmb_test", stop, torch.device("cuda", index))
    assert devices() == 0


def test_status_is_read_on_its_device(devices, monkeypatch):
    class Lib:
        @staticmethod
        def vmb_device_status(stream, out):
            out._obj.value = 10 * devices() + stream
            return 0
    monkeypatch.setattr(N, "lib", Lib)
    assert N.device_status(torch.device("cuda", 1)) == 111 and N.device_status(torch.device("cuda", 0)) == 100


def test_every_call_with_a_stream_goes_through_launch():
    """No module calls an entry that takes a stream by itself."""
    for path in Path(N.__file__).parent.glob("*.py"):
        if path.name != "_native.py":
            direct = set(re.findall(r"N\.lib\.(vmb_\w+)\(", path.read_text()))
            assert {n for n in direct if not n.endswith("_bytes")} <= {"vmb_kernel_launches"}, path.name
