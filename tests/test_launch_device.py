"""Weight preparation and the operators beside the layer launch on the device that holds the tensors, whichever is
the current one: a null stream means the current device's. On the CPU, with the
library and the tensors stood in for."""
import contextlib
import types

import pytest
import torch

from netra_moe import layers
from netra_moe import weights as W


class Tensor:
    is_cuda = True

    def __init__(self, shape, dtype, device):
        self.shape, self.dtype, self.device = shape, dtype, device

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 20

    def numel(self):
        return 1 << 20

    def element_size(self):
        return 1


@pytest.fixture
def launches(monkeypatch):
    """(entry point, current device, stream's device) of every call into the library."""
    current, calls = [0], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], torch.device(d).index
        yield
        current[0] = before

    class Library:
        def __getattr__(self, name):
            def call(*args):
                calls.append((name, current[0], args[-1]))
                return 0
            return call

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: types.SimpleNamespace(cuda_stream=torch.device(d).index))
    monkeypatch.setattr(torch, "empty", lambda shape, dtype, device: Tensor(shape, dtype, device))
    monkeypatch.setattr(torch, "empty_like", lambda t: Tensor(t.shape, t.dtype, t.device))
    monkeypatch.setattr(W, "bridge_library", Library)
    monkeypatch.setattr(layers, "_raw_stream", lambda index: index)
    return calls


@pytest.mark.parametrize("index", [0, 1])
def test_every_entry_point_launches_on_the_tensors_device(launches, index):
    dev = torch.device("cuda", index)
    W.quantize_blocks(Tensor((1, 128, 128), torch.float32, dev))
    q = Tensor((1, 128, 128), torch.uint8, dev)
    for gate_up in (False, True):
        W.pack_tiles(q, gate_up)
        W.pack_tiles_from_aiter(q, gate_up)
    W.device_copy(q, Tensor((1, 128, 128), torch.uint8, dev))
    assert {n for n, _, _ in launches} == {
        "netra_moe_quant_blocks", "netra_moe_pack_tiles", "netra_moe_pack_tiles_gate_up", "netra_moe_pack_tiles_from_aiter",
        "netra_moe_pack_tiles_gate_up_from_aiter", "netra_moe_copy"}
    assert {(d, s) for _, d, s in launches} == {(index, index)}


@pytest.mark.parametrize("index", [0, 1])
def test_operators_launch_on_the_tensors_device(launches, index):
    layers.launch(W.bridge_library().netra_linear_forward, "netra_linear_forward", torch.device("cuda", index), 1, 2)
    assert launches == [("netra_linear_forward", index, index)] and torch.cuda.current_device() == 0
