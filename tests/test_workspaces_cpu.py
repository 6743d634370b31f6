"""Workspaces that callers give: an empty tensor, whose null pointer would turn a call into a question for the size, is refused, and
so is one on another device."""
import ctypes

import pytest
import torch

import tcu_scope_amd.binding as b


class Entry:
    """Stands for a C entry point with a two-phase workspace; remembers its calls."""

    __name__ = "entry"

    def __init__(self, workspace_at, need):
        self.workspace_at, self.need, self.calls = workspace_at, need, []

    def __call__(self, *args):
        self.calls.append(args)
        ws = args[self.workspace_at]
        if not (ws.value if isinstance(ws, ctypes.c_void_p) else ws):
            args[self.workspace_at + 1]._obj.value = self.need
        return 0

    def ran(self):
        return any((a[self.workspace_at].value if isinstance(a[self.workspace_at], ctypes.c_void_p) else a[self.workspace_at]) for a in self.calls)


CPU = torch.device("cpu")


def test_recurrent_block_calls():
    entry = Entry(0, 512)
    with pytest.raises(ValueError, match="empty"):
        b._call_with_workspace(entry, (), (1,), torch.empty(0, dtype=torch.uint8), CPU, None)
    with pytest.raises(ValueError, match="contiguous tensor on"):
        b._call_with_workspace(entry, (), (1,), torch.empty(512, dtype=torch.uint8, device="meta"), CPU, None)
    assert not entry.calls
    b._call_with_workspace(entry, (), (1,), torch.empty(128, dtype=torch.float32), CPU, None)
    assert entry.ran() and entry.calls[-1][1]._obj.value == 512
    b._workspace_sizes.clear()


def test_full_array_calls(monkeypatch):
    monkeypatch.setattr(b, "_stream", lambda stream: None)
    x = torch.zeros(8, dtype=torch.float16)
    entry = Entry(3, 512)
    with pytest.raises(ValueError, match="empty"):
        b._workspace(entry, x, x, 8, 0, 0, 0, torch.empty(0, dtype=torch.uint8), None)
    with pytest.raises(ValueError, match="contiguous tensor on"):
        b._workspace(entry, x, x, 8, 0, 0, 0, torch.empty(512, dtype=torch.uint8, device="meta"), None)
    assert not entry.ran()
    b._workspace(entry, x, x, 8, 0, 0, 0, torch.empty(512, dtype=torch.uint8), None)
    assert entry.ran()
    nothing = Entry(3, 0)  # a call that needs none takes an empty one
    b._workspace(nothing, x, x, 0, 0, 0, 0, torch.empty(0, dtype=torch.uint8), None)
    assert len(nothing.calls) == 2


@pytest.mark.parametrize("name", ["scan", "reduce"])
def test_by_key_calls(monkeypatch, name):
    entry = Entry(5 if name == "scan" else 7, 512)
    monkeypatch.setattr(b, "_stream", lambda stream: None)
    monkeypatch.setattr(b, "_need_f16", lambda t, name: None)
    monkeypatch.setattr(b, "_key_bits", lambda keys: 32)
    monkeypatch.setattr(b, "lib", lambda: type("L", (), {f"tcu_seg_{name}_by_key_f16": entry})())
    x, keys = torch.zeros(8, dtype=torch.float16), torch.zeros(8, dtype=torch.int32)
    call = b.seg_scan_by_key if name == "scan" else b.seg_reduce_by_key
    with pytest.raises(ValueError, match="empty"):
        call(keys, x, workspace=torch.empty(0, dtype=torch.uint8))
    with pytest.raises(ValueError, match="contiguous tensor on"):
        call(keys, x, workspace=torch.empty(512, dtype=torch.uint8, device="meta"))
    assert not entry.ran()
    call(keys, x, workspace=torch.empty(512, dtype=torch.uint8))
    assert entry.ran()
