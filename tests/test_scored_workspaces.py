"""CPU: what the calls of scored attention, and of the preference and policy losses, hand the library as workspaces: the size
that it asks for, by the place each signature has for it, and a buffer of that size. Sizes are ones that no shape has."""
from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch

from mlx_train_perf import _native
from mlx_train_perf.attention import api as attn_api
from mlx_train_perf.core import preference as P

SIZES = {"mtp_attn_scored_fwd_workspace_bytes": 4160, "mtp_attn_scored_bwd_workspace_bytes": 4224, "mtp_attn_scored_plan_bytes": 4288,
         "mtp_attn_scored_fwd_f32_workspace_bytes": 4352, "mtp_attn_scored_bwd_f32_workspace_bytes": 4416,
         "mtp_pref_workspace_bytes": 4480, "mtp_policy_workspace_bytes": 4544}


class _FakeLib:
    """Entry points that note their arguments, after what their signatures make of them."""

    def __init__(self, sizes):
        self.sizes, self.calls = sizes, {}

    def __getattr__(self, name):
        kinds = _native.SIGNATURES[name][1]
        if name in self.sizes:
            return lambda *a: (len(a) == len(kinds) or pytest.fail(name)) and self.sizes[name]

        def call(*a):
            assert len(a) == len(kinds), name
            for kind, x in zip(kinds, a):
                kind(x)
            self.calls[name] = a
            return 0
        return call


@pytest.fixture
def run(monkeypatch):
    """run(sizes, f): the calls that f makes, and the sizes in bytes of the buffers that it allocates, by address."""
    def go(sizes, f):
        lib, made = _FakeLib(sizes), {}
        real = torch.empty

        def empty(*a, **kw):
            t = real(*a, **kw)
            made[t.data_ptr()] = t.numel() * t.element_size()
            keep.append(t)
            return t

        keep: list[torch.Tensor] = []   # so that no address is used twice
        with monkeypatch.context() as m:
            m.setattr(_native, "on_device", lambda t: contextlib.nullcontext())
            m.setattr(_native, "load", lambda: lib)
            m.setattr(_native, "stream_of", lambda t: 77)
            m.setattr(torch, "empty", empty)
            f()
        return lib.calls, made
    return go


def _workspace(calls, made, name, size):
    """The last three of every launching entry point: workspace, its size, the stream."""
    ws, bytes_, stream = calls[name][-3:]
    assert _native.SIGNATURES[name][1][-2:] == [ctypes.c_size_t, ctypes.c_void_p]
    assert bytes_ == size and stream == 77, name
    assert ws is None if size == 0 else made[ws] == size, name


@pytest.mark.parametrize("spans", [False, True])
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize(("dtype", "suffix"), [(torch.bfloat16, ""), (torch.float32, "_f32")])
def test_scored_attention(run, dtype, suffix, split, spans):
    sizes = dict(SIZES)
    if not split:
        sizes["mtp_attn_scored_fwd_workspace_bytes"] = sizes["mtp_attn_scored_fwd_f32_workspace_bytes"] = 0
    b, s, hq, hkv, dh = 1, 8, 2, 1, 64
    end = torch.arange(1, s + 1, dtype=torch.int32)[None] if spans else None
    start = torch.zeros_like(end) if spans else None

    def step():
        q = torch.zeros(b, hq, s, dh, dtype=dtype, requires_grad=True)
        k = torch.zeros(b, hkv, s, dh, dtype=dtype)
        o = attn_api._ScoredAttention.apply(q, k, k, None, start, end, 0.125, not spans, 5.0)[0]
        o.sum().backward()

    calls, made = run(sizes, step)
    fwd, bwd = f"mtp_attn_scored_fwd{suffix}", f"mtp_attn_scored_bwd{suffix}"
    assert set(calls) == {fwd, bwd}
    for name in (fwd, bwd):
        _workspace(calls, made, name, sizes[f"{name}_workspace_bytes"])
    # the shape, and the spans, where the signatures have them
    assert calls[fwd][3:8] == (b, hq, hkv, s, dh) and calls[fwd][12:14] == (_native.ptr(start), _native.ptr(end))
    at = 8 if dtype == torch.bfloat16 else 6
    assert calls[bwd][at:at + 5] == (b, hq, hkv, s, dh) and calls[bwd][at + 9:at + 11] == (_native.ptr(start), _native.ptr(end))
    if dtype == torch.bfloat16:   # the forward's low bits and plan are the backward's
        low, plan = calls[fwd][15:17]
        assert made[plan] == sizes["mtp_attn_scored_plan_bytes"] if spans else plan is None
        assert calls[bwd][4] == low is not None and calls[bwd][5] == plan


def test_preference(run):
    x = torch.zeros(4, 3, requires_grad=True)
    calls, made = run(SIZES, lambda: P._Preference.apply(x, torch.zeros(4, 3), None, None, 2, 0, 0.1, 0.0, 1)[0].backward())
    assert set(calls) == {"mtp_pref_fwd", "mtp_pref_bwd"}
    _workspace(calls, made, "mtp_pref_fwd", SIZES["mtp_pref_workspace_bytes"])


def test_policy(run):
    x = torch.zeros(4, 3, requires_grad=True)
    calls, made = run(SIZES, lambda: P._Policy.apply(x, torch.zeros(4, 3), None, torch.zeros(4), None, None, 4, 0.2, 0.2, 0.0, 1)[0].backward())
    assert set(calls) == {"mtp_policy_fwd", "mtp_policy_bwd"}
    _workspace(calls, made, "mtp_policy_fwd", SIZES["mtp_policy_workspace_bytes"])
