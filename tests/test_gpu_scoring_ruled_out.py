"""Tokens that are ruled out: a logit of -inf, from a weight of -inf or from a finite product past fp32's range. Their probability is
0 and so is what they add to an entropy, a divergence or a gradient."""
from __future__ import annotations

import math

import _scoring as S
import pytest
import torch

from mlx_train_perf import DenseHead, distillation_loss, token_logprobs
from mlx_train_perf.core import scoring

pytestmark = pytest.mark.gpu

_CASES = [(3, 72, "bf16"), (17, 64, "bf16"), (40, 72, "bf16"), (90, 64, "bf16"), (140, 72, "bf16"), (140, 64, "bf16"),
          (3, 36, "fp32"), (40, 64, "fp32"), (140, 36, "fp32"), (140, 33, "fp32")]
_OUT = (8, 31, 299)


def _make(n, d, dtype, weight):
    hidden, hd, w = S.make(n, d, 300, dtype=dtype, seed=5)
    hidden[:, 5] = 2.0
    w[_OUT, 5] = weight
    w = w.to(hidden.dtype)
    return hidden, DenseHead(weight=w.cuda().requires_grad_(True), trainable=True), w.double()


@pytest.mark.parametrize("targets", [False, True])
@pytest.mark.parametrize(("n", "d", "dtype"), _CASES)
def test_entropy_of_infinite_weights(n, d, dtype, targets):
    hidden, hd, w = _make(n, d, dtype, -math.inf)
    y = torch.arange(n) % 8 if targets else None
    for top in (0, 5):
        with torch.no_grad():
            got = token_logprobs(hidden.cuda(), hd, None if y is None else y.cuda(), top=top)
        logp = torch.log_softmax(hidden.double() @ w.T, 1)
        want = torch.special.entr(logp.exp()).sum(1)
        S.within(got.entropy, want, S.stat(300) + 256 * S.U + 128 * S.stat(300), "entropy")
        if targets:
            S.within(got.logprobs, logp.gather(1, y[:, None])[:, 0], S.stat(300) + 256 * S.U, "logprobs")


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize(("n", "d", "dtype"), _CASES)
def test_gradients_of_products_past_the_range(n, d, dtype, keep, monkeypatch):
    if not keep:
        monkeypatch.setattr(scoring, "_kept_bytes", lambda x: 0)
    hidden, hd, w = _make(n, d, dtype, -3e38)
    h = hidden.cuda().requires_grad_(True)
    halves = keep and n <= 128
    clean, live = hidden.double(), torch.ones(n, dtype=torch.bool)
    y = torch.arange(n) % 8
    z = S.logits(hidden, w, live)
    logprobs, entropy, _, _ = S.score(z, y, live, 1.0, 0)
    got = token_logprobs(h, hd, y.cuda())
    S.within(got.entropy, entropy, S.stat(300) + 256 * S.U + 128 * S.stat(300), "entropy")
    a, b = torch.randn(2, n, generator=torch.Generator().manual_seed(n))
    p = torch.softmax(z.detach(), 1)
    for outs, want, cts, size in (((got.logprobs,), logprobs * a.double(), (a,), a.abs()),
                                  ((got.logprobs, got.entropy), logprobs * a.double() + entropy * b.double(), (a, b), a.abs() + 64 * b.abs())):
        (gz,) = torch.autograd.grad(want.sum(), z, retain_graph=True)
        grad = torch.autograd.grad(outs, (h, hd.weight), [x.cuda() for x in cts], retain_graph=True)
        dh, dh_off, dw, dw_off = S.gradient_bounds(gz, p, size.double(), clean, w, True, dtype, halves)
        S.within(grad[0], dh, dh_off, "d_hidden")
        S.within(grad[1], dw, dw_off, "d_weight")


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize(("n", "d", "dtype"), _CASES)
def test_distillation(n, d, dtype, keep, monkeypatch):
    """Off the list; and on it, where forward's divergence is infinite and the others' term is 0."""
    if not keep:
        monkeypatch.setattr(scoring, "_kept_bytes", lambda x: 0)
    hidden, hd, w = _make(n, d, dtype, -3e38)
    h = hidden.cuda().requires_grad_(True)
    g = torch.Generator().manual_seed(n)
    ids = torch.stack([torch.randperm(300, generator=g)[:9] for _ in range(n)])
    ids[torch.isin(ids, torch.tensor(_OUT))] = -1
    listed = ids.clone()
    listed[:, 3] = 31
    lp = (torch.log_softmax(torch.randn(n, 9, generator=g), 1) - 0.5).float()
    for kind, of in (("forward", ids), ("reverse", ids), ("reverse", listed), ("jsd", ids), ("jsd", listed)):
        args = {"kind": kind, "beta": 0.4, "temperature": 1.0, "renormalize": False, "reduction": "none"}
        z = S.logits(hidden, w, torch.ones(n, dtype=torch.bool))
        want, _ = S.distill(z, of, lp, None, **args)
        got = distillation_loss(h, hd, of.cuda(), lp.cuda(), **args)
        S.within(got, want, 64 * (S.stat(300) + 256 * S.U), f"loss, {kind}")
        ct = torch.randn(n, generator=g)
        (gz,) = torch.autograd.grad(want, z, ct.double())
        grad = torch.autograd.grad(got, (h, hd.weight), ct.cuda())
        dh, dh_off, dw, dw_off = S.gradient_bounds(gz, torch.softmax(z.detach(), 1), 64 * ct.abs().double(), hidden.double(), w, True, dtype,
                                                   keep and n <= 128)
        S.within(grad[0], dh, dh_off, f"d_hidden, {kind}")
        S.within(grad[1], dw, dw_off, f"d_weight, {kind}")


@pytest.mark.parametrize("n", [3, 140])
def test_a_target_that_is_ruled_out(n):
    """Log probability -inf; its gradient's column is the incoming gradient and nothing of the entropy's."""
    hidden, hd, w = _make(n, 64, "bf16", -3e38)
    h = hidden.cuda().requires_grad_(True)
    got = token_logprobs(h, hd, torch.full((n,), 8, device="cuda"))
    assert bool((got.logprobs == -math.inf).all())
    z = S.logits(hidden, w, torch.ones(n, dtype=torch.bool))
    logp, entropy, _, _ = S.score(z, torch.full((n,), 8), torch.ones(n, dtype=torch.bool), 1.0, 0)
    p = torch.softmax(z.detach(), 1)
    for b in (0.0, 0.3):
        (gz,) = torch.autograd.grad((logp + b * entropy).sum(), z, retain_graph=True)
        (dw,) = torch.autograd.grad((got.logprobs, got.entropy), (hd.weight,), (torch.ones(n, device="cuda"), torch.full((n,), b, device="cuda")),
                                    retain_graph=True)
        _, _, want, off = S.gradient_bounds(gz, p, torch.full((n,), 1 + 64 * b, dtype=torch.float64), hidden.double(), w, True,
                                            "bf16", n <= 128)
        S.within(dw, want, off, "d_weight")
