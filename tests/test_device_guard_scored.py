"""CPU: the calls of scored attention and of the preference and policy losses run with their tensors' device current
(as test_device_guard.py holds for the others), each with what the library asks for as workspace."""
from __future__ import annotations

import contextlib

import pytest
import torch

from mlx_train_perf import _native
from mlx_train_perf.attention import api as attn_api
from mlx_train_perf.core import preference as P


class _FakeLib:
    """Every entry point notes its name, the current device and its arguments; a workspace is 64 bytes."""

    def __init__(self, state: dict):
        self.state, self.calls = state, []

    def __getattr__(self, name):
        if name.endswith("workspace_bytes"):
            return lambda *a: 64

        def call(*a):
            self.calls.append((name, self.state["dev"]))
            assert 64 in a or name in ("mtp_attn_scored_fwd", "mtp_pref_bwd", "mtp_policy_bwd")
            return 0
        return call


@pytest.fixture
def fake(monkeypatch):
    state = {"dev": "cuda:7"}   # the caller's current device is not the tensors'
    lib = _FakeLib(state)

    @contextlib.contextmanager
    def device(dev):
        prev, state["dev"] = state["dev"], torch.device(dev)
        try:
            yield
        finally:
            state["dev"] = prev

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(_native, "load", lambda: lib)
    monkeypatch.setattr(_native, "stream_of", lambda t: 0)
    return lib


def _ran(fake, device, *names):
    assert fake.calls == [(name, device) for name in names]


@pytest.mark.parametrize(("dtype", "suffix"), [(torch.bfloat16, ""), (torch.float32, "_f32")])
def test_scored_attention(fake, dtype, suffix):
    q = torch.zeros(1, 2, 8, 64, dtype=dtype, requires_grad=True)
    k = torch.zeros(1, 1, 8, 64, dtype=dtype)
    o = attn_api._ScoredAttention.apply(q, k, k, None, None, None, 0.125, True, 5.0)[0]
    o.sum().backward()
    _ran(fake, q.device, f"mtp_attn_scored_fwd{suffix}", f"mtp_attn_scored_bwd{suffix}")


def test_preference(fake):
    x = torch.zeros(4, 3, requires_grad=True)
    P._Preference.apply(x, torch.zeros(4, 3), None, None, 2, 0, 0.1, 0.0, 1)[0].backward()
    _ran(fake, x.device, "mtp_pref_fwd", "mtp_pref_bwd")


def test_policy(fake):
    x = torch.zeros(4, 3, requires_grad=True)
    P._Policy.apply(x, torch.zeros(4, 3), None, torch.zeros(4), None, None, 4, 0.2, 0.2, 0.0, 1)[0].backward()
    _ran(fake, x.device, "mtp_policy_fwd", "mtp_policy_bwd")
