"""CPU tests of calls that clipping refuses or takes: what was refused has changed nothing, the tensors' versions among it, and
outputs that hold their values in the tensors' order are taken."""

import pytest
import torch

from symmetrix import node_ops


@pytest.fixture
def on_device(monkeypatch):
    """Tensors pass for ones of the device, so that a call goes as far as the C boundary."""
    monkeypatch.setattr(node_ops, "_stream", lambda device: 0)


def test_refused_calls_change_no_version(on_device):
    """What the C boundary refuses, before any launch, is not seen as changed by a graph that kept it."""
    a, b = torch.ones(8), torch.ones(8)
    for call, text in ((lambda: node_ops.clip_gradients([a, a], 1.0), "two outputs overlap"),
                       (lambda: node_ops.clip_gradients([a, b], 1.0, out=[b, a]), "not its own"),
                       (lambda: node_ops.clip_gradients([a], -1.0), "max_norm"),
                       (lambda: node_ops.clip_gradients([a], 1.0, scale=0.0), "scale"),
                       (lambda: node_ops.clip_gradients([a], 1.0, scale=-1.0, out=[b]), "scale")):
        with pytest.raises(ValueError, match=text):
            call()
    assert a._version == b._version == 0


def test_outputs_in_the_tensors_order(monkeypatch):
    """An axis of one value has any stride: what counts is the order of the values."""
    calls = []
    monkeypatch.setattr(node_ops, "_stream", lambda device: calls.append(device) or 0)
    monkeypatch.setattr(node_ops.lib, "smx_clip_gradients", lambda *args: 0)
    turned = torch.ones(4, 1, 3).transpose(0, 2)  # [3][1][4], strides 1, 3, 3
    other = torch.empty_strided((3, 1, 4), (1, 77, 3))
    assert not turned.is_contiguous() and turned.stride() != other.stride()
    for to in (other, torch.empty_strided((3, 4), (1, 3)), torch.empty_strided((1, 3, 4), (5, 1, 3))):
        node_ops.clip_gradients([turned], 1.0, out=[to])
    assert len(calls) == 3
    for bad in (torch.ones(3, 1, 4), torch.ones(12), torch.ones(4, 3).t().contiguous()):
        with pytest.raises(ValueError, match="strides"):
            node_ops.clip_gradients([turned], 1.0, out=[bad])
    assert len(calls) == 3
