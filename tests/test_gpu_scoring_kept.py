"""What a scoring or distillation call holds on to: logits only for a backward that hidden states or a trainable weight get, in both
autograd paths; and which path takes a call."""
from __future__ import annotations

import _scoring as S
import pytest
import torch

from mlx_train_perf import DenseHead, _native, distillation_loss, token_logprobs

pytestmark = pytest.mark.gpu

_N, _V = 200, 3200
_KEPT = _N * _V * 4


@pytest.fixture(params=[True, False], ids=["nodes", "functions"])
def path(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(_native, "_nodes", False)
    assert (_native.nodes() is not None) == request.param


def _held(call, peak=False):
    """Bytes that a call's results hold, or (peak) the call at its most."""
    call()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    held = (torch.cuda.max_memory_allocated() if peak else torch.cuda.memory_allocated()) - before
    del out
    return held


@pytest.mark.parametrize("loss", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_logits_are_kept_for_a_gradient_alone(path, dtype, loss):
    hidden, hd, _ = S.make(_N, 64, _V, dtype=dtype)
    w = hd.weight.cuda()
    ids, lp, _ = (x.cuda() for x in S.teacher_list(_N, _V, 4, holes=False))
    y = torch.zeros(_N, dtype=torch.int64, device="cuda")

    def held(hidden_asks, weight_asks, trainable, grad=True):
        h = hidden.cuda().requires_grad_(hidden_asks)
        head = DenseHead(weight=w.detach().requires_grad_(weight_asks), trainable=trainable)
        with torch.set_grad_enabled(grad):
            return _held((lambda: distillation_loss(h, head, ids, lp)) if loss else (lambda: token_logprobs(h, head, y)), peak=not grad)

    assert held(True, False, False) >= _KEPT and held(False, True, True) >= _KEPT
    assert held(True, False, False, grad=False) < _KEPT // 4
    assert held(False, True, True, grad=False) < _KEPT // 4
    assert held(False, False, False) < _KEPT // 4
    assert held(False, True, False) < _KEPT // 4   # a frozen head's weight gets no gradient, whatever it asks for


@pytest.mark.parametrize("n", [20, 200])
def test_without_a_graph_both_paths_give_the_same_bits(n, monkeypatch):
    """A hidden state that asks for a gradient, under no_grad."""
    hidden, hd, _ = S.make(n, 64, _V, seed=2)
    h, hd = hidden.cuda().requires_grad_(True), S.to(hd, "cuda")
    ids, lp, _ = (x.cuda() for x in S.teacher_list(n, _V, 4, holes=False))
    y = torch.arange(n, device="cuda")

    @torch.no_grad()
    def run():
        return [*token_logprobs(h, hd, y, top=3), distillation_loss(h, hd, ids, lp, reduction="none")]

    nodes = run()
    monkeypatch.setattr(_native, "_nodes", False)
    assert all(torch.equal(a, b) for a, b in zip(run(), nodes, strict=True))
