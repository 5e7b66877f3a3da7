"""Every operator makes its tensors' device the current one while it calls the
library: kernels are launched on the current device, whatever their pointers
say.  On the CPU, with a library and devices that only take notes."""
import contextlib

import pytest
import torch

import rdna2_ops._native as nat

DEVICE = torch.device("cpu", 1)  # allocates here, and has an index


class Anywhere:
    """A device that every tensor is on."""

    index = 1

    def __eq__(self, other):
        return True


class Notes:
    """Stands for the library and for CUDA's current device."""

    def __init__(self, current):
        self.current, self.calls = current, []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, self.current, args[-1] if args else None))
            return 256 if name.endswith("bytes") else 0
        return call

    @contextlib.contextmanager
    def device(self, device):
        before, self.current = self.current, getattr(device, "index", device)
        yield
        self.current = before


@pytest.fixture(params=[0, 1], ids=["another device", "this device"])
def notes(request, monkeypatch):
    notes = Notes(request.param)
    monkeypatch.setattr(nat, "library", lambda: notes)
    monkeypatch.setattr(nat, "require_device", lambda *tensors: DEVICE)
    monkeypatch.setattr(nat, "eager_only", lambda *tensors: None)
    monkeypatch.setattr(nat, "stream_ptr", lambda device: 1000 + device.index)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: notes.current)
    monkeypatch.setattr(torch.cuda, "device", notes.device)
    before = notes.current
    yield notes
    assert notes.current == before
    launches = [call for call in notes.calls if not call[0].endswith("bytes")]
    assert launches and all(call[1:] == (1, 1001) for call in launches), notes.calls


def _names(notes):
    return [call[0] for call in notes.calls]


def test_rotary(notes, monkeypatch):
    from rdna2_ops.rotary import rotary
    monkeypatch.setattr(nat, "require_device", lambda *tensors: Anywhere())
    rotary(torch.zeros(2, 1, 64), torch.zeros(4, 64), torch.arange(2))
    assert _names(notes) == ["b2_rotary"]


def test_append(notes, monkeypatch):
    from rdna2_ops import kv_cache
    monkeypatch.setattr(nat, "require_device", lambda *tensors: Anywhere())
    cache = kv_cache.PagedKVCache(3, 2, 64, page_size=16, device="cpu")
    x, table = torch.zeros(2, 2, 64), torch.zeros(2, 1, dtype=torch.int32)
    cache.append(x, x, torch.ones(2, dtype=torch.int32), table, q=x, angles=torch.zeros(4, 64))
    assert _names(notes) == ["b2_kv_append"]


def test_attend_and_read(notes):
    from rdna2_ops import kv_cache
    kv_cache._workspace_bytes.cache_clear()
    cache = kv_cache.PagedKVCache(3, 2, 64, page_size=16, device="cpu")
    table = torch.zeros(2, 1, dtype=torch.int32)
    cache.attend(torch.zeros(2, 2, 64).half(), torch.ones(2, dtype=torch.int32), table, return_lse=True)
    cache.read(table[0])
    kv_cache._workspace_bytes.cache_clear()
    assert _names(notes) == ["b2_kv_attention_workspace_bytes", "b2_kv_attention", "b2_kv_read"]
    assert notes.calls[0][1] == 1  # it goes by the device's multiprocessors


def test_quantized_linears(notes, monkeypatch):
    from rdna2_ops import _args, qlinear
    monkeypatch.setattr(_args, "fp32_vector", lambda *args, **kw: None)  # would compare devices
    w = torch.zeros(32, 64, dtype=torch.int8)
    qlinear.act_quant(torch.zeros(2, 64))
    qlinear.w8a8_linear(torch.zeros(2, 64), w, torch.ones(32))
    assert [n for n in _names(notes) if not n.endswith("bytes")] == ["b2_act_quant", "b2_quant_linear"]


def test_every_launch_goes_by_its_device():
    """No wrapper takes a stream by itself, but those of a process that has one device."""
    from conftest import PKG
    for path in sorted((PKG / "rdna2_ops").glob("*.py")):
        if path.name not in ("_native.py", "column_parallel.py"):
            text = path.read_text().replace("stream = nat.stream_ptr(dev)", "")  # a workspace's key
            assert "stream_ptr" not in text, path.name
