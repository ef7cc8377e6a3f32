"""Targets that have nearly all of the mass: log p, and 1 - p in the gradient at the target, are right to the digits of 1 and not to
those of a logit.

Logits near 430 that are exact (_shifted), and ordinary ones of many terms (_many_terms). u = 2^-24. log p = x_y - m - log2 s in the log2 domain,
with the target's own logit among the sums: x_y - m is rounded once, below u; s is 1 and a little, summed in chains of at most 64 additions
after the largest term (16 + 2 of a lane's tile, its tiles, the joins of lanes, waves, splits), and its logarithm and their difference
are rounded: 72 u of 1. What s has beside 1, 1 - p, is off by a relative `rel`: stat(V) + 256 u, the rounding of exponents of up to 1024 in size
(2 * 1024 u) and, for logits of d terms, twice their own d u |h||w|."""
from __future__ import annotations

import _scoring as S
import pytest
import torch

from mlx_train_perf import DenseHead, token_logprobs
from mlx_train_perf.core import scoring

pytestmark = pytest.mark.gpu


def _shifted(n, v, dtype):
    g = torch.Generator().manual_seed(n)
    hidden, w = S.grid(g, n, 64), S.grid(g, v, 64) / 4
    y = 37 * n % v            # every token's, 8 to 19 above the others
    hidden[:, :32], w[:, :32] = 15.5, 0.875
    hidden[:, 32:40] = 1 + (torch.arange(n) % 16)[:, None] * 3 / 32
    w[:, 32:40] = 0
    w[y, 32:40] = 1.0
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    return hidden.to(dt), w.to(dt), torch.full((n,), y)


def _many_terms(n, v, dtype):
    g, d = torch.Generator().manual_seed(n), 1024
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    w = (torch.randn(v, d, generator=g) / 16).to(dt)
    y = torch.randint(0, v, (n,), generator=g)
    mine = w[y].double()
    hidden = torch.randn(n, d, generator=g) + mine * (torch.linspace(12, 26, n)[:, None] / mine.square().sum(1, keepdim=True))
    return hidden.to(dt), w, y


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("make", [_shifted, _many_terms])
@pytest.mark.parametrize(("n", "top"), [(5, 0), (40, 3), (100, 0), (300, 0), (300, 4)])
def test_targets(n, top, make, dtype, keep, monkeypatch):
    if not keep:
        monkeypatch.setattr(scoring, "_kept_bytes", lambda x: 0)
    v = 1500
    hidden, w, y = make(n, v, dtype)
    h = hidden.cuda().requires_grad_(True)
    hd = DenseHead(weight=w.cuda().requires_grad_(True), trainable=True)
    got = token_logprobs(h, hd, y.cuda(), top=top)
    z = hidden.double() @ w.double().T
    logp = torch.log_softmax(z, 1)
    lp = logp.gather(1, y[:, None])[:, 0]
    left = logp.exp().scatter(1, y[:, None], 0.0).sum(1)
    assert float(left.min()) < (2e-4 if n > 16 else 0.1)
    size = (hidden.double().abs() @ w.double().abs().T).amax(1)
    rel = S.stat(v) + 256 * S.U + 2048 * S.U + (0 if make is _shifted else 2 * 1024 * S.U * size)
    off = 72 * S.U + left * rel + 4 * S.U * lp.abs()
    S.within(got.logprobs, lp, off, "logprobs")
    if top:
        assert torch.equal(got.top_ids[:, 0].cpu(), z.argmax(1))
        first = got.top_ids[:, 0].cpu() == y
        assert torch.equal(got.top_logprobs[:, 0].cpu()[first], got.logprobs.detach().cpu()[first])
    a = torch.randn(n, generator=torch.Generator().manual_seed(1)).double()
    p = logp.exp()
    hot = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
    gz = a[:, None] * torch.where(hot > 0, left[:, None], -p)
    halves = dtype == "bf16" and keep and n <= 128
    step = (S.R * S.R if halves else S.R) if dtype == "bf16" else S.U
    g_off = a.abs()[:, None] * torch.where(hot > 0, off[:, None], p * (rel + 2048 * S.U if make is _shifted else rel[:, None] + 2048 * S.U)) + step * gz.abs()
    dh, dw = torch.autograd.grad(got.logprobs, (h, hd.weight), a.float().cuda())
    half = S.R if dtype == "bf16" else S.U
    for got_, g, go, m in ((dh, gz, g_off, w.double()), (dw, gz.T, g_off.T, hidden.double())):
        want = g @ m
        bound = go @ m.abs() + 2 * g.shape[1] * S.U * (g.abs() @ m.abs()) + half * want.abs() + 1e-12
        S.within(got_, want, bound, "gradient")
