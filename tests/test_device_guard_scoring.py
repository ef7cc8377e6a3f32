"""CPU: the calls of token scoring and distillation run with their tensors' device current (as test_device_guard.py holds for the
loss and attention), each with what the library asks for as workspace, and hand the kept logits on."""
from __future__ import annotations

import contextlib

import pytest
import torch

from mlx_train_perf import _native
from mlx_train_perf.core import scoring


class _FakeLib:
    """Every launching entry point notes its name, the current device and its arguments; a workspace is 64 bytes."""

    def __init__(self, state: dict):
        self.state, self.calls = state, []

    def __getattr__(self, name):
        if name.endswith("workspace_bytes"):
            return lambda *a: 64
        if name.endswith(("chunk", "row_block")):
            return lambda *a: 256

        def call(*a):
            self.calls.append((name, self.state["dev"], a))
            assert 64 in a
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
    monkeypatch.setenv("MTP_LCE_TRANSPOSED_HEAD", "0")
    kept = []
    room = scoring._kept_logits
    monkeypatch.setattr(scoring, "_kept_logits", lambda x: kept.append(room(x)) or kept[-1])
    lib.kept = kept
    return lib


def _inputs(dtype, trainable):
    hidden = torch.zeros(4, 64, dtype=dtype, requires_grad=True)
    w = torch.zeros(100, 64, dtype=dtype, requires_grad=trainable)
    return scoring._Inputs(hidden, w, None, None, None, _native.HEAD_DENSE, w)


@pytest.mark.parametrize("trainable", [False, True])
@pytest.mark.parametrize(("dtype", "suffix"), [(torch.bfloat16, ""), (torch.float32, "_f32")])
class TestCalls:
    def _ran(self, fake, x, *names):
        assert [(name, dev) for name, dev, _ in fake.calls] == [(name, x.hidden.device) for name in names]
        assert len(fake.kept) == 1 and fake.kept[0].numel() == 4 * 128
        for _, _, args in fake.calls:
            assert fake.kept[0].data_ptr() in args
        assert x.hidden.grad is not None and (x.w.grad is not None) == x.w.requires_grad

    def test_scoring(self, fake, dtype, suffix, trainable):
        x = _inputs(dtype, trainable)
        out = scoring._TokenLogprobs.apply(*x, torch.zeros(4, dtype=torch.int64), -100, 3, 1.0)
        (out[0].sum() + out[1].sum()).backward()
        self._ran(fake, x, f"mtp_logprobs_fwd{suffix}", f"mtp_logprobs_bwd{suffix}")

    def test_distillation(self, fake, dtype, suffix, trainable):
        x = _inputs(dtype, trainable)
        scoring._Distillation.apply(*x, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2), None, 0, 0.5, 1.0, 0, 1).backward()
        self._ran(fake, x, f"mtp_distill_fwd{suffix}", f"mtp_distill_bwd{suffix}")


def test_nothing_is_kept_without_a_backward(fake):
    x = _inputs(torch.float32, False)
    scoring._TokenLogprobs.apply(*x._replace(hidden=x.hidden.detach()), None, -100, 0, 1.0)
    assert not fake.kept and [c[0] for c in fake.calls] == ["mtp_logprobs_fwd_f32"]
