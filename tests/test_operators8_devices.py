"""CPU: the size of a workspace is asked with the tensors' device current, and kept by device."""

from __future__ import annotations

import contextlib

import pytest


class _Machine:
    """Two devices of unlike numbers of CUs; an entry answers for the current one, as the library's do."""

    def __init__(self):
        self.current, self.asked = 0, []

    def __getattr__(self, name):
        def entry(*args):
            self.asked.append((name, self.current))
            return 1000 + 100 * self.current + len(args)

        return entry

    @contextlib.contextmanager
    def device(self, index):
        before, self.current = self.current, index
        yield
        self.current = before


@pytest.mark.parametrize("module,args", [("adapters", (64, 3, 8192, 16, 2, 64, False)), ("mxfp8", (200, 128, 16384, False)),
                                         ("mxfp4", (200, 128, 16384, False, True))])
def test_sizes_go_by_the_device(monkeypatch, module, args):
    import importlib

    import torch

    from minimal_inference_amd import _lib

    size = importlib.import_module(f"minimal_inference_amd.{module}")._workspace_size
    machine = _Machine()
    size.cache_clear()
    try:
        with monkeypatch.context() as m:
            m.setattr(_lib, "load", lambda: machine)
            m.setattr(torch.cuda, "device", machine.device)
            m.setattr(torch._C, "_cuda_getDevice", lambda: machine.current, raising=False)
            assert [size(*args, d) - size(*args, 0) for d in (0, 1, 1, 0)] == [0, 100, 100, 0]
            machine.current = 1  # what was asked before stays
            assert size(*args, 0) + 100 == size(*args, 1) and machine.current == 1
            assert [d for _, d in machine.asked] == [0, 1]
    finally:
        size.cache_clear()
