"""CPU check: the token mixers' entries launch with their tensors' device current, whichever device the caller has.

No GPU is touched: the tensors are fake ones of ``cuda:1``, the library is a stand-in that notes which device was current
at each call, and ``torch.cuda``'s device functions are replaced by ones that keep a number.
"""
import contextlib
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


class Library:
    """Answers every entry with success (sizes with 1024 bytes) and notes the device that was current."""

    def __init__(self, machine):
        self.machine, self.calls = machine, []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, self.machine.current))
            return 1024 if name.endswith("_bytes") else 0
        return entry

    def launches(self):
        return [(name, device) for name, device in self.calls if not name.endswith("_bytes")]


class Machine:
    """Two devices, the first one current, with the default stream (handle 0) on both."""

    def __init__(self, monkeypatch):
        from reax_engine_runtime_v3_b200 import _native
        self.current, self.switches = 0, 0
        self.library = Library(self)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)
        monkeypatch.setattr(torch.cuda, "device", self.device)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        monkeypatch.setattr(_native, "load", lambda: self.library)
        monkeypatch.setattr(_native, "_current_device", lambda: self.current)
        monkeypatch.setattr(_native, "_raw_stream", lambda index: 0)
        monkeypatch.setattr(_native, "_workspaces", {})

    @contextlib.contextmanager
    def device(self, device):
        index = device if isinstance(device, int) else torch.device(device).index
        before, self.current = self.current, index
        self.switches += 1
        try:
            yield
        finally:
            self.current = before


def calls(device):
    """One call of every entry, by name, on fake tensors of `device`."""
    from reax_engine_runtime_v3_b200 import gated_delta
    from reax_engine_runtime_v3_b200.kv_int8 import Int8Cache
    new = lambda *shape, dtype=torch.bfloat16: torch.empty(shape, dtype=dtype, device=device)
    ints = lambda *shape: new(*shape, dtype=torch.int32)
    floats = lambda *shape: new(*shape, dtype=torch.float32)
    cache = Int8Cache.empty(4, 2, 64, 16, device)
    gdn = new(3, 1, 64), new(3, 1, 64), new(3, 2, 64), floats(3, 2), floats(3, 2), floats(3, 2, 64, 64)
    return {
        "reax_gdn_prefill": lambda: gated_delta.prefill(*gdn),
        "reax_gdn_decode": lambda: gated_delta.decode(*gdn),
        "reax_kv8_append": lambda: cache.append(new(3, 2, 64), new(3, 2, 64), ints(3, 2), ints(3)),
        "reax_kv8_read": lambda: cache.read(ints(3, 2), ints(3), ints(4), 5),
        "reax_kv8_attend": lambda: cache.attend(new(3, 4, 64), ints(3, 2), ints(3)),
    }


@pytest.mark.parametrize("entry", ["reax_gdn_prefill", "reax_gdn_decode", "reax_kv8_append", "reax_kv8_read", "reax_kv8_attend"])
@pytest.mark.parametrize("index", [0, 1])
def test_entries_launch_on_their_tensors_device(monkeypatch, entry, index):
    with FakeTensorMode(), warnings.catch_warnings():
        warnings.simplefilter("ignore")                      # (a fake tensor's address is 0, with a warning)
        call = calls(f"cuda:{index}")[entry]
        machine = Machine(monkeypatch)
        call()
    assert machine.library.launches() == [(entry, index)]
    assert machine.current == 0
    if index == 0:
        assert machine.switches == 0                         # the usual call pays for no switch


def test_status_is_read_on_the_device_asked_for(monkeypatch):
    from reax_engine_runtime_v3_b200 import _native
    machine = Machine(monkeypatch)
    assert _native.mixer_status() == 0 and _native.mixer_status(device=torch.device("cuda", 1)) == 0
    assert machine.library.launches() == [("reax_mixer_status", 0), ("reax_mixer_status", 1)] and machine.current == 0
