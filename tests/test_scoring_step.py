"""Scoring and distillation through the trainer adapters on a tiny random-init model (CPU): a teacher's lists into a student's
step, against plain logits; positions left out; refusals; and (with a stand-in for the library) the device and the
workspaces of the calls."""
from __future__ import annotations

import contextlib

import pytest
import torch

from mlx_train_perf import DenseHead, QuantizedHead, _native
from mlx_train_perf.adapters.transformers_lm import make_distillation_loss_fn, make_token_logprobs_fn
from mlx_train_perf.core import scoring
from mlx_train_perf.errors import AdapterError
from tests.test_adapters import _tiny_llama
from tests.test_preference_step import _batch, _mask


def _logp(model, batch, temperature=1.0):
    return torch.log_softmax(model(input_ids=batch[:, :-1]).logits.double() / temperature, -1)


def test_scores():
    m = _tiny_llama(seed=0)
    batch, lengths = _batch(3, 9)
    with torch.no_grad():
        got = make_token_logprobs_fn(m, top=5, temperature=1.5, impl="naive")(m, batch, lengths)
        logp = _logp(m, batch, 1.5)
    keep = _mask(lengths, 9)
    want = logp.gather(-1, batch[:, 1:, None])[..., 0]
    assert torch.allclose(got.logprobs.double(), torch.where(keep, want, 0.0), atol=1e-5)
    assert torch.allclose(got.entropy.double(), torch.where(keep, -(logp.exp() * logp).sum(-1), 0.0), atol=1e-5)
    value, ids = logp.topk(5, -1)
    assert torch.equal(got.top_ids[keep], ids[keep]) and bool((got.top_ids[~keep] == -1).all())
    assert torch.allclose(got.top_logprobs[keep].double(), value[keep], atol=1e-5)


@pytest.mark.parametrize("kind", ["forward", "reverse", "jsd"])
def test_a_student_learns_a_teachers_scores(kind):
    m, teacher = _tiny_llama(seed=0), _tiny_llama(seed=1)
    batch, lengths = _batch(3, 9)
    with torch.no_grad():
        lists = make_token_logprobs_fn(teacher, top=12, impl="naive")(teacher, batch)
    loss = make_distillation_loss_fn(m, kind=kind, beta=0.3, impl="naive")(m, batch, lengths, lists.top_ids, lists.top_logprobs)
    loss.backward()
    grad = m.model.layers[0].self_attn.q_proj.weight.grad.clone()
    m.zero_grad()
    keep = _mask(lengths, 9)
    with torch.no_grad():
        t = _logp(teacher, batch).topk(12, -1)
        lt = torch.cat([t.values, (1 - t.values.exp().sum(-1, keepdim=True)).log()], -1)
    lq = _logp(m, batch).gather(-1, t.indices)
    lq = torch.cat([lq, (1 - lq.exp().sum(-1, keepdim=True)).log()], -1)
    lm = torch.log(0.3 * lt.exp() + 0.7 * lq.exp())
    rows = {"forward": (lt.exp() * (lt - lq)).sum(-1), "reverse": (lq.exp() * (lq - lt)).sum(-1),
            "jsd": 0.3 * (lt.exp() * (lt - lm)).sum(-1) + 0.7 * (lq.exp() * (lq - lm)).sum(-1)}[kind]
    want = rows[keep].mean()
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5 * max(1.0, abs(float(want.detach())))
    want.backward()
    assert torch.allclose(grad, m.model.layers[0].self_attn.q_proj.weight.grad, atol=1e-6)


def test_refusals():
    m = _tiny_llama()
    m.config.final_logit_softcapping = 30.0
    for make in (make_token_logprobs_fn, make_distillation_loss_fn):
        with pytest.raises(AdapterError, match="final_logit_softcapping"):
            make(m)
    m.config.final_logit_softcapping = None
    batch, _ = _batch(2, 5)
    with pytest.raises(AdapterError, match="enable_flash_attention"):
        make_token_logprobs_fn(m, impl="naive")(m, batch, spans=object())


class _FakeLib:
    """Every entry point notes its name, the current device and its arguments; sizes are 64."""

    def __init__(self, state):
        self.state, self.calls = state, []

    def __getattr__(self, name):
        if name.endswith("_bytes") or name.endswith("_chunk") or name.endswith("_block"):
            return lambda *a: 64

        def call(*a):
            self.calls.append((name, self.state["dev"]))
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
    monkeypatch.setattr(_native, "load", lambda: lib)
    monkeypatch.setattr(_native, "stream_of", lambda t: 0)
    monkeypatch.setattr(scoring._loss, "_transposed_head", lambda *a: None)
    return lib


@pytest.mark.parametrize(("dtype", "suffix"), [(torch.bfloat16, ""), (torch.float32, "_f32")])
@pytest.mark.parametrize("kind", ["trainable", "frozen", "q4"])
def test_calls_run_with_their_tensors_device_current(fake, dtype, suffix, kind):
    h = torch.zeros(3, 64, dtype=dtype, requires_grad=True)
    if kind == "q4":
        sb = torch.zeros(8, 1, dtype=torch.bfloat16)
        head = QuantizedHead(w_q=torch.zeros(8, 8, dtype=torch.int32), scales=sb, biases=sb)
    else:
        head = DenseHead(weight=torch.zeros(8, 64, dtype=dtype, requires_grad=True), trainable=kind == "trainable")
    x = scoring._inputs(h, head)
    y = torch.zeros(3, dtype=torch.int64)
    parts = scoring._TokenLogprobs.apply(*x, y, -100, 2, 1.0)
    (parts[0].sum() + parts[1].sum()).backward()
    ids = torch.zeros(3, 2, dtype=torch.int64)
    scoring._Distillation.apply(*x, ids, torch.zeros(3, 2), None, 0, 0.5, 1.0, 0, 1).backward()
    names = ["mtp_logprobs_fwd", "mtp_logprobs_bwd", "mtp_distill_fwd", "mtp_distill_bwd"]
    assert fake.calls == [(name + suffix, torch.device("cpu")) for name in names]
    if kind == "trainable":
        assert head.weight.grad is not None and head.weight.grad.shape == (8, 64)
    assert h.grad.dtype is dtype
