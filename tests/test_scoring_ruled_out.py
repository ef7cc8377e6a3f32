"""The reference impl with tokens that a weight of -inf rules out: they add 0 to an entropy, a divergence and their gradients."""
from __future__ import annotations

import math

import pytest
import torch

from mlx_train_perf import DenseHead, distillation_loss, token_logprobs


def _heads():
    """A head with rows of -inf, and the head without them."""
    g = torch.Generator().manual_seed(1)
    hidden, w = torch.rand(5, 8, generator=g, dtype=torch.float64) + 0.1, torch.randn(12, 8, generator=g, dtype=torch.float64)
    ruled = torch.cat([w, torch.full((2, 8), -math.inf, dtype=torch.float64)])
    return hidden, w, ruled


def test_entropy():
    hidden, w, ruled = _heads()
    y = torch.arange(5)
    a, b = (token_logprobs(hidden, DenseHead(weight=x), y, top=12, impl="reference") for x in (w, ruled))
    assert torch.allclose(a.entropy, b.entropy, atol=1e-13) and torch.allclose(a.logprobs, b.logprobs, atol=1e-13)
    assert torch.equal(a.top_ids, b.top_ids)
    grads = []
    for x in (w, ruled):
        x = x.clone().requires_grad_(True)
        r = token_logprobs(hidden, DenseHead(weight=x, trainable=True), y, impl="reference")
        grads += torch.autograd.grad(r.entropy.sum() + r.logprobs.sum(), x)
    assert torch.allclose(grads[0], grads[1][:12], atol=1e-13) and bool((grads[1][12:] == 0).all())


@pytest.mark.parametrize("kind", ["reverse", "jsd"])
def test_on_the_list(kind):
    """The teacher's mass there is the student's 0; only jsd notices that the rest has less of it."""
    hidden, _, ruled = _heads()
    ids = torch.tensor([0, 3, 12, 5]).expand(5, 4)
    lp = torch.log_softmax(torch.arange(4.0).double(), 0).expand(5, 4) - 0.3
    x = ruled.clone().requires_grad_(True)
    got = distillation_loss(hidden, DenseHead(weight=x, trainable=True), ids, lp, kind=kind, reduction="none", impl="reference")
    logp = torch.log_softmax(hidden @ ruled.T, 1)
    q, t = logp[:, ids[0]].exp(), lp.exp()
    q, t = (torch.cat([p, 1 - p.sum(1, keepdim=True)], 1) for p in (q, t))
    kl = lambda a, b: torch.where(a > 0, a * (a / b).log(), 0.0).sum(1)   # noqa: E731
    want = kl(q, t) if kind == "reverse" else 0.5 * kl(t, (t + q) / 2) + 0.5 * kl(q, (t + q) / 2)
    assert torch.allclose(got, want, atol=1e-12)
    (g,) = torch.autograd.grad(got.sum(), x)
    assert bool(torch.isfinite(g).all()) and bool((g[12:] == 0).all())
