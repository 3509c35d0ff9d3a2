"""Workspace sizes that depend on the number of SMs are asked for where the tensors are, and kept for that device alone."""
from __future__ import annotations

import contextlib
import types

import pytest
import torch

SIZES = {0: 592, 1: 1024}  # of two devices with other numbers of SMs


@pytest.fixture
def two_devices(monkeypatch):
    from comfy_kitchen.backends import cuda as backend

    state = types.SimpleNamespace(current=0, calls=[])

    @contextlib.contextmanager
    def on_device(device):
        before, state.current = state.current, device.index
        yield
        state.current = before

    class Library:
        def __getattr__(self, name):
            return lambda *_: SIZES[state.current]

        def ck_clip_grad_norm(self, grads, counts, dtypes, n, max_norm, norm, ws, need, stream):
            state.calls.append((state.current, need))
            return 0 if need >= SIZES[state.current] else 1

        def ck_last_error(self):
            return b"workspace too small"

    lib, empty = Library(), torch.empty
    monkeypatch.setattr(backend, "_lib", lib)
    monkeypatch.setattr(backend, "load_library", lambda: lib)
    monkeypatch.setattr(backend, "_on_device", on_device)
    monkeypatch.setattr(backend, "_stream", lambda device: 0)
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: empty(*a, **kw))
    backend._workspace_bytes.cache_clear()
    yield backend, state
    backend._workspace_bytes.cache_clear()


def _gradient(index):
    memory = torch.zeros(8)
    return types.SimpleNamespace(device=torch.device("cuda", index), dtype=torch.float32, layout=torch.strided, is_contiguous=lambda: True,
                                 data_ptr=memory.data_ptr, numel=memory.numel, memory=memory)


def test_clipping_on_either_device(two_devices):
    backend, state = two_devices
    for index in (0, 1, 0, 1):
        backend.clip_grads([_gradient(index)], 1.0)
    assert state.calls == [(i, SIZES[i]) for i in (0, 1, 0, 1)]


def test_sizes_are_kept_by_device(two_devices):
    backend, state = two_devices
    for name in ("ck_rms_norm_backward_workspace_bytes", "ck_layer_norm_backward_workspace_bytes", "ck_scaled_mm_workspace_bytes"):
        for index in (0, 1, 0):
            with backend._on_device(torch.device("cuda", index)):
                assert backend._workspace_bytes(name, 2, 4, 64, device=index) == SIZES[index]
