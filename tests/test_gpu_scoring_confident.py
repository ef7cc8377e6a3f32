"""Distillation of students that give nearly all of their mass to the teacher's list: what it leaves of 1, R, is small, and its
logarithm (forward, jsd, reverse) and T / R (forward's gradient) are right to R's own digits.

The logits are exact (tests/_scoring.py) and up to 45. With u = 2^-24, a probability's relative error, R's among them, is
rel = stat(V) + 256 u: log2(e) / temperature is one fp32 number in every term, off by u of itself, so differences of exponents
(below 64) are off by 64 u; a term's own exponent (below 92 in the log2 domain) is rounded once, 64 u, and its exponential is off
by 2 u; the sums are stat(V); lifting partial sums to a common maximum adds 64 + 2 u. None of it grows as 1 / R. The loss is off by
rel times its derivatives by the log probabilities, taken here one by one, and by its rounding. A gradient by a logit, p (f_R - F) off the
list and q (f - F) on it, is off by rel times p (64 + 2 T / R) and q 64: f_R is -T / R or a logarithm below 32 with the error of one, F
a mean of such."""
from __future__ import annotations

import math

import _scoring as S
import pytest
import torch

from mlx_train_perf import DenseHead, distillation_loss
from mlx_train_perf.core import scoring

pytestmark = pytest.mark.gpu


def _confident(n, v, k, *, dtype, seed):
    """(hidden, head, weights in fp64, ids, log probabilities): the list's logits stand 0 to 32 above the others'."""
    d, g = 64, torch.Generator().manual_seed(seed)
    hidden, w = S.grid(g, n, d), S.grid(g, v, d) / 4
    ids = torch.randperm(v, generator=g)[:k]
    hidden[:, :16] = ((torch.arange(n) + 1) / n * 127).round()[:, None] / 32
    w[:, :16] = 0
    w[ids, :16] = 0.5
    hidden[:, 16:24], w[:, 16:24] = 2.0, 0.5
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    _, lp, _ = S.teacher_list(n, v, k, seed=seed, holes=False)
    ids = torch.stack([ids[torch.randperm(k, generator=g)] for _ in range(n)])
    return hidden.to(dt), w.double(), ids, lp, DenseHead(weight=w.to(dt).cuda(), trainable=False)


def _loss(lq, lrq, lt, rt, kind, beta):
    """Per row, from the log probabilities alone."""
    t, q = lt.exp(), lq.exp()
    if kind == "forward":
        return (t * (lt - lq)).sum(1) + rt * (rt.log() - lrq)
    if kind == "reverse":
        return (q * (lq - lt)).sum(1) + lrq.exp() * (lrq - rt.log())
    m, rm = (beta * t + (1 - beta) * q).log(), (beta * rt + (1 - beta) * lrq.exp()).log()
    return (beta * t * (lt - m) + (1 - beta) * q * (lq - m)).sum(1) + beta * rt * (rt.log() - rm) + (1 - beta) * lrq.exp() * (lrq - rm)


def _check(n, v, k, dtype, temperature, kind, *, grads, halves, seed):
    beta = 0.4
    hidden, w, ids, lp, hd = _confident(n, v, k, dtype=dtype, seed=seed)
    z = (hidden.double() @ w.T).requires_grad_(True)
    # R as a sum of its own
    logp = torch.log_softmax(z / temperature, 1)
    off_list = torch.ones(n, v, dtype=torch.bool).scatter_(1, ids, False)
    lr = torch.logsumexp(logp.masked_fill(~off_list, -math.inf), 1)
    r = lr.detach().exp()
    assert float(r.min()) < (1e-6 if temperature < 1.5 else 1e-4)
    lrq = lr + (r.clamp(min=S.TAIL).log() - r.log())
    lrq = torch.where(r < S.TAIL, (lr.exp() + (S.TAIL - r)).log(), lrq)   # the floor leaves the gradient of what it lifts
    lt = lp.double()
    rt = (1 - lt.exp().sum(1)).clamp(min=S.TAIL)
    lq = logp.gather(1, ids)
    want = _loss(lq, lrq, lt, rt, kind, beta)
    free = [x.detach().requires_grad_(True) for x in (lq, lrq)]
    by_lq, by_lr = torch.autograd.grad(_loss(*free, lt, rt, kind, beta).sum(), free)
    rel = S.stat(v) + 256 * S.U
    h = hidden.cuda().requires_grad_(grads)
    got = distillation_loss(h, hd, ids.cuda(), lp.cuda(), kind=kind, beta=beta, temperature=temperature, reduction="none")
    S.within(got, want, rel * (by_lq.abs().sum(1) + by_lr.abs()) + 4 * S.U * (1 + want.detach().abs()), f"loss, {kind}")
    if not grads:
        return
    ct = torch.randn(n, generator=torch.Generator().manual_seed(seed + 1), dtype=torch.float64).float()
    (gz,) = torch.autograd.grad(want, z, ct.double())
    (got_dh,) = torch.autograd.grad(got, h, ct.cuda())
    size = torch.where(off_list, (64 + 2 * rt / r.clamp(min=S.TAIL))[:, None], 64.0)
    p = logp.detach().exp() * size * ct.double().abs()[:, None] / temperature
    dh, off, _, _ = S.gradient_bounds(gz, p, torch.ones(n, dtype=torch.float64), hidden.double(), w, False, dtype, halves)
    S.within(got_dh, dh, off, f"d_hidden, {kind}")


@pytest.mark.parametrize("temperature", [0.7, 1.0, 1.7, 2.0])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize(("n", "v", "k"), [(5, 1000, 50), (16, 700, 128), (40, 20011, 100), (64, 1000, 1), (200, 1000, 50), (300, 3001, 128)])
def test_lists_with_nearly_all_of_the_mass(n, v, k, dtype, temperature):
    """Few tokens; and many, whose forward keeps its logits."""
    for kind in ("forward", "reverse", "jsd"):
        _check(n, v, k, dtype, temperature, kind, grads=True, halves=n <= 128, seed=n)


@pytest.mark.parametrize("temperature", [0.7, 1.7])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize(("n", "v", "k"), [(200, 1000, 50), (300, 3001, 128), (40, 1000, 50)])
def test_logits_that_are_not_kept(n, v, k, dtype, temperature, monkeypatch):
    monkeypatch.setattr(scoring, "_kept_bytes", lambda x: 0)
    for kind in ("forward", "reverse", "jsd"):
        _check(n, v, k, dtype, temperature, kind, grads=True, halves=False, seed=n)
        _check(n, v, k, dtype, temperature, kind, grads=False, halves=False, seed=n)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [3, 150])
def test_the_whole_vocabulary_is_listed(n, dtype):
    """Nothing is off the list: its sum is empty, the rest is the floor."""
    v, dt = 100, torch.bfloat16 if dtype == "bf16" else torch.float32
    g = torch.Generator().manual_seed(n)
    hidden, w = S.grid(g, n, 64), S.grid(g, v, 64) / 4
    ids = torch.arange(v).expand(n, v)
    lp = torch.log_softmax(torch.randn(n, v, generator=g), 1) - 0.25
    got = distillation_loss(hidden.to(dt).cuda(), DenseHead(weight=w.to(dt).cuda(), trainable=False), ids.cuda(), lp.cuda(), reduction="none")
    lt, lq = lp.double(), torch.log_softmax(hidden.double() @ w.double().T, 1)
    rt = 1 - lt.exp().sum(1)
    want = (lt.exp() * (lt - lq)).sum(1) + rt * (rt / S.TAIL).log()
    S.within(got, want, 2 * (S.stat(v) + 256 * S.U) + 4 * S.U * (1 + want.abs()), "loss")
