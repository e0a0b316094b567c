"""The binding's way onto a device and stream, with torch's side of it replaced."""
import contextlib

import pytest
import torch

from helixml_b200 import _lib as L
from helixml_b200 import ops


@pytest.mark.parametrize("current", [0, 1])
def test_calls_run_on_the_operands_device(current, monkeypatch):
    """On the stream torch uses on the operands' device, which is made the current one for the call and only for it."""
    seen, now = [], [current]

    @contextlib.contextmanager
    def device(dev):
        before, now[0] = now[0], dev
        yield
        now[0] = before

    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 1000 + dev, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)

    def fn(*args):
        seen.append((now[0], *args))
        return 0

    ops._call(1, fn, "a", 7)
    assert seen == [(1, "a", 7, 1001)] and now == [current]
    with pytest.raises(L.HxError):
        ops._call(1, lambda *a: 10)
    assert now == [current]
