"""Which autograd path takes a scoring or distillation call: the C++ nodes those whose every tensor is plain, the Python Functions
the others; and both ask for a gradient on the same calls."""
from __future__ import annotations

import _scoring as S
import pytest
import torch
from torch.autograd import forward_ad

from mlx_train_perf import DenseHead, QuantizedHead, _native, distillation_loss, token_logprobs
from mlx_train_perf.core import scoring


class _Marked(torch.Tensor):
    pass


def _tensors(device="cpu"):
    hidden, hd, _ = S.make(6, 64, 40, dtype="fp32", seed=1)
    ids, lp, mask = S.teacher_list(6, 40, 3, holes=False)
    return hidden.to(device), S.to(hd, device), ids.to(device), lp.to(device), mask.to(device)


def test_every_tensor_of_a_call_decides(monkeypatch):
    monkeypatch.setattr(_native, "nodes", lambda: "nodes")
    hidden, hd, ids, lp, mask = _tensors()
    x = scoring._inputs(hidden, hd)
    y = torch.zeros(6, dtype=torch.int64)
    assert scoring._nodes(x, y, -100, 3, 1.0) == "nodes" and scoring._nodes(x, None) == "nodes"
    assert scoring._nodes(x, ids, lp, mask, 0, 0.5) == "nodes" and scoring._nodes(x, ids, lp, None) == "nodes"
    assert scoring._nodes(x, y.as_subclass(_Marked), -100, 3, 1.0) is None
    for i in range(3):
        others = [t.as_subclass(_Marked) if i == j else t for j, t in enumerate((ids, lp, mask))]
        assert scoring._nodes(x, *others) is None
    with forward_ad.dual_level():
        assert scoring._nodes(x, ids, forward_ad.make_dual(lp, torch.ones_like(lp)), mask) is None
        assert scoring._nodes(x, ids, lp, mask) == "nodes"


def test_the_reference_impl_has_a_teachers_tangent():
    """In forward mode; a backward to it is refused, as before."""
    hidden, hd, ids, lp, _ = _tensors()
    hidden, hd = hidden.double(), DenseHead(weight=hd.weight.double())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(lp.double(), torch.full((6, 3), 0.01, dtype=torch.float64))
        loss = distillation_loss(hidden, hd, ids, dual, impl="reference")
        tangent = forward_ad.unpack_dual(loss).tangent
    up, down = (distillation_loss(hidden, hd, ids, lp.double() + 0.01 * s, impl="reference") for s in (1e-4, -1e-4))
    assert abs(float(tangent) - float(up - down) / 2e-4) < 1e-6


@pytest.mark.gpu
def test_a_teachers_tangent_is_refused():
    hidden, hd, ids, lp, _ = _tensors("cuda")
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        distillation_loss(hidden, hd, ids, forward_ad.make_dual(lp, torch.ones_like(lp)))


@pytest.mark.gpu
def test_subclasses_give_the_same_values():
    hidden, hd, ids, lp, mask = _tensors("cuda")
    y = torch.arange(6, device="cuda")
    assert torch.equal(token_logprobs(hidden, hd, y.as_subclass(_Marked)).logprobs.as_subclass(torch.Tensor), token_logprobs(hidden, hd, y).logprobs)
    want = distillation_loss(hidden, hd, ids, lp, mask=mask)
    for i in range(3):
        a, b, c = (t.as_subclass(_Marked) if i == j else t for j, t in enumerate((ids, lp, mask)))
        assert torch.equal(distillation_loss(hidden, hd, a, b, mask=c).as_subclass(torch.Tensor), want)


@pytest.mark.gpu
@pytest.mark.parametrize("asks", [(), ("hidden",), ("scales",), ("biases",), ("hidden", "scales")])
@pytest.mark.parametrize("nodes", [True, False])
def test_a_4bit_heads_scales_and_biases(asks, nodes, monkeypatch):
    """They are inputs of the call like hidden, and get no gradient."""
    if not nodes:
        monkeypatch.setattr(_native, "_nodes", False)
    hidden, hd, _ = S.make(6, 64, 40, head="q4", dtype="bf16", seed=1)
    t = {"hidden": hidden, "scales": hd.scales, "biases": hd.biases}
    t = {k: x.cuda().requires_grad_(k in asks) for k, x in t.items()}
    head = QuantizedHead(w_q=hd.w_q.cuda(), scales=t["scales"], biases=t["biases"])
    ids, lp, _ = (x.cuda() for x in S.teacher_list(6, 40, 3, holes=False))
    for out in (token_logprobs(t["hidden"], head).entropy.sum(), distillation_loss(t["hidden"], head, ids, lp)):
        assert out.requires_grad == bool(asks)
        if not asks:
            continue
        grads = torch.autograd.grad(out, list(t[k] for k in asks), allow_unused=True)
        assert all((g is not None) == (k == "hidden") for k, g in zip(asks, grads))


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [True, False])
def test_results_can_be_changed_in_place(nodes, monkeypatch):
    """What a call hands out is not what its backward reads; of the entropy, which it does read, autograd says so."""
    if not nodes:
        monkeypatch.setattr(_native, "_nodes", False)
    hidden, hd, _, _, _ = _tensors("cuda")
    y = torch.arange(6, device="cuda")

    def grad(change):
        h = hidden.clone().requires_grad_(True)
        r = token_logprobs(h, hd, y, top=2)
        logprobs = change(r.logprobs)
        r.top_logprobs.zero_()
        r.top_ids.zero_()
        return torch.autograd.grad(logprobs.sum() + r.entropy.sum(), h)[0]

    assert torch.equal(grad(lambda x: x.mul_(2.0)), grad(lambda x: x * 2.0))
    h = hidden.clone().requires_grad_(True)
    entropy = token_logprobs(h, hd, y).entropy
    entropy.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        entropy.sum().backward()
