"""CPU checks of the Python side of decay attention and layer norm, with the library and the
device queries replaced: what buffers a call makes, which calls it refuses, and what autograd
is told."""
import types

import pytest
import torch

from atlas_b200 import scan


@pytest.fixture
def host(monkeypatch):
    """No device: one stream, which captures while ``host.capturing`` is set."""
    from atlas_b200 import decay_attention, layer_norm
    h = types.SimpleNamespace(capturing=False)
    for m in (scan, decay_attention, layer_norm):
        monkeypatch.setattr(m, "away", lambda dev: False)
        monkeypatch.setattr(m, "stream_of", lambda dev: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: h.capturing)
    return h


def test_captured_scratch_is_the_graphs_own(host):
    """A captured call's address is replayed for as long as the graph lives: its scratch is neither
    a buffer that a later, larger call replaces nor one that another call or graph uses."""
    ws, dev = scan.Workspace(), torch.device("cpu")
    eager, _ = ws.get(100, dev)
    host.capturing = True
    a, n = ws.get(50, dev)
    b, _ = ws.get(50, dev)
    assert n >= 50 and a.numel() >= 50
    assert len({x.data_ptr() for x in (eager, a, b)}) == 3
    assert ws.get(0, dev) == (None, 0)
    host.capturing = False
    assert ws.get(80, dev)[0] is eager
    larger, n = ws.get(200, dev)
    assert n >= 200 and larger is not eager and ws.get(200, dev)[0] is larger
