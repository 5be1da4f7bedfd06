"""The host layers of the operators around the attention without a GPU: CPU
tensors pass for the GPU's, the library is a stand-in, and a test sees each call
at the moment of its launch."""
import ctypes
import gc

import pytest
import torch

from ops_amd import _host, _lib, cache, rope, tree


class Library:
    """Workspace sizes are 64 bytes; every other entry is only named."""

    def __getattr__(self, name):
        return (lambda *a: 64) if name.endswith("workspace_size") else name


def live(address):
    """Whether some tensor that is still held owns the address."""
    for t in gc.get_objects():
        if issubclass(type(t), torch.Tensor):
            s = t.untyped_storage()
            if s.data_ptr() <= address < s.data_ptr() + max(s.nbytes(), 1):
                return True
    return False


def addresses(args):
    """(name, address) of everything that a call hands to the library."""
    for i, a in enumerate(args):
        if isinstance(a, int) and a >= 1 << 20:  # (counts and sizes here are smaller)
            yield f"argument {i}", a
        for name, kind in getattr(getattr(a, "_obj", None), "_fields_", ()):
            v = getattr(a._obj, name)
            if name == "pools":
                pools = ctypes.cast(v, ctypes.POINTER(_lib.CachePool))
                for k in range(a._obj.npools):
                    yield f"pool {k}", pools[k].base
            elif kind is ctypes.c_void_p and v:
                yield name, v


@pytest.fixture
def launches(monkeypatch):
    """The calls made: (entry, arguments, tensors' addresses that nobody held any more)."""
    seen = []

    def call(device, fn, *args):
        seen.append((fn, args, [n for n, at in addresses(args) if not live(at)]))

    for m in (_host, rope, tree, cache):
        monkeypatch.setattr(m, "need_gpu", lambda name, t, device=None: None)
        if m is not _host:
            monkeypatch.setattr(m, "call", call)
    monkeypatch.setattr(_lib, "load", Library)
    return seen
