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
        before, self.current = self.current, device.index
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
    assert notes.calls and all(call[1] == 1 for call in notes.calls), notes.calls
    assert all(call[2] == 1001 for call in notes.calls if not call[0].endswith("bytes")), notes.calls


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
