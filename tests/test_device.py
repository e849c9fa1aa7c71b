"""Which stream a call goes to when its tensors lie on another device than the current one (host only)."""
import pytest
import torch

from kq import ops


@pytest.mark.parametrize("current,index,handle,fine", [(0, 0, 0, True), (1, 1, 0, True), (0, 1, 64, True), (0, 1, 0, False),
                                                       (2, 0, 0, False)])
def test_a_default_stream_is_its_own_devices(monkeypatch, current, index, handle, fine):
    monkeypatch.setattr(ops, "_raw_stream", lambda i: handle)
    monkeypatch.setattr(ops, "_current", lambda: current)
    monkeypatch.setattr(ops, "_several", True)
    if fine:
        assert ops._stream(torch.device("cuda", index)) == handle
    else:
        with pytest.raises(ValueError, match="cuda:%d must be the current device" % index):
            ops._stream(torch.device("cuda", index))
